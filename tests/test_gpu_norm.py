"""RMS norm, its codes and its gradient.

The forward is fixed by its steps: h rounded to the rows' type, the mean in 64 bits, r rounded to fp32, two
fp32 products, the codes of fp32 rows.  So every output is compared bit for bit.  (r itself would differ
where 1 / sqrt(mean + eps) falls within the 64-bit sum's error, some 2^-50, of a border between two fp32
numbers: one row in 2^25.)

The gradient's sums are fp32.  With u = 2^-24, the mean of d xh is off by at most n u of its magnitudes, n the
additions one after the other: at most 64 in a thread up to K = 2^16, 6 in a wave and 16 of waves.  An element
of dx adds 8 roundings of its terms, one of dgain the M rows' and 64 of the partial sums'.
"""
import numpy as np
import pytest

import mx
import tier_amd
from mx import FORMATS, MxRows
from rows import TINY, TYPES, UNIT, Rows, f32, from_bits, to_bits
from test_gpu_i8 import quantize
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, F16, BF16 = tier_amd.F32, tier_amd.F16, tier_amd.BF16
U, EPS = 2.0 ** -24, np.float32(1e-5)


def rows(M, K, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((M, K)) * spread).astype(np.float32)
    x[:, 7::61] *= 11
    return x


def gains(K, seed=0):
    return (1 + 0.2 * np.random.default_rng(seed).standard_normal(K)).astype(np.float32)


def forward(t, x, res, g, eps=EPS):
    """(h, r, y) by the definition: x and res fp32 values of the type."""
    x = x.astype(np.float32)
    h = x if res is None else from_bits(t, to_bits(t, x + res.astype(np.float32))).astype(np.float32)
    with np.errstate(all="ignore"):
        r = (1.0 / np.sqrt((h.astype(np.float64) ** 2).mean(1) + np.float64(eps))).astype(np.float32)
        return h, r, ((h * r[:, None]).astype(np.float32) * g).astype(np.float32)


SIZES = [(1, 1, 0, 0), (3, 127, 0, 1), (2, 128, 3, 0), (5, 1408, 0, 0), (1, 5120, 0, 0), (2, 5121, 2, 3), (3, 8192, 0, 0),
         (2, 16389, 0, 0), (1, 40000, 8, 8), (515, 300, 1, 0), (520, 2048, 0, 0), (513, 5120, 0, 0), (513, 9000, 0, 4)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,pad,skip", SIZES)
def test_forward(gpu, t, M, K, pad, skip):
    X, R = Rows(t, M, K, rows(M, K, 1), pad, skip), Rows(t, M, K, rows(M, K, 2, 2.0), pad + 1, skip)
    g = gains(K)
    for res in (None, R):
        h, r, y = forward(t, X.values(), None if res is None else res.values(), g)
        H, Y = Rows(t, M, K, None, pad, skip), Rows(t, M, K, None, pad + 2, skip)
        rb = tier_amd.i8_row_bytes(K) + (16 if pad else 0)
        Q, S, RS = hip.DeviceBuffer(M * rb + 16), f32(np.full(M + 1, 7.0)), f32(np.full(M + 1, 7.0))
        Q.fill_bytes(0x55)
        tier_amd.rms_norm(X.ptr, t, X.ld, res and res.ptr, R.ld, f32(g).ptr, EPS, H.ptr, H.ld, Y.ptr, Y.ld, Q.ptr, rb, S.ptr,
                          RS.ptr, M, K)
        hip.synchronize()
        assert np.array_equal(H.bits(), to_bits(t, h)) and np.array_equal(Y.bits(), to_bits(t, y))
        assert np.array_equal(RS.download(np.float32), np.append(r, np.float32(7)))
        q, s = quantize(y)
        got, need = Q.download(np.int8)[:M * rb].reshape(M, rb), tier_amd.i8_row_bytes(K)
        assert np.array_equal(got[:, :K], q) and not got[:, K:need].any() and (got[:, need:] == 0x55).all()
        assert (Q.download(np.int8)[M * rb:] == 0x55).all()
        assert np.array_equal(S.download(np.float32), np.append(s, np.float32(7)))
        assert H.outside_kept() and Y.outside_kept() and X.outside_kept()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,pad,skip", SIZES)
def test_forward_mx(gpu, fmt, t, M, K, pad, skip):
    X, R = Rows(t, M, K, rows(M, K, 3), pad, skip), Rows(t, M, K, rows(M, K, 4, 2.0), 0, 1)
    g, Q, Y = gains(K, 1), MxRows(fmt, M, K, pad=pad), Rows(t, M, K)
    tier_amd.rms_norm_mx(X.ptr, t, X.ld, R.ptr, R.ld, f32(g).ptr, EPS, None, 0, Y.ptr, K, fmt, Q.q.ptr, Q.rb, Q.s.ptr, Q.sb,
                         None, M, K)
    hip.synchronize()
    _, _, y = forward(t, X.values(), R.values(), g)
    c, s = Q.get()
    want, scales = mx.quantize(fmt, y)
    assert np.array_equal(s, scales) and np.array_equal(c, want) and np.array_equal(Y.bits(), to_bits(t, y))


@pytest.mark.parametrize("K", [640, 33000])
@pytest.mark.parametrize("which", ["y", "q", "h", "rstd"])
def test_each_output_alone(gpu, which, K):
    M, t = 4, BF16
    X, R, g = Rows(t, M, K, rows(M, K, 5)), Rows(t, M, K, rows(M, K, 6)), gains(K)
    h, r, y = forward(t, X.values(), R.values(), g)
    rb, O, S = tier_amd.i8_row_bytes(K), Rows(t, M, K), f32(np.zeros(M))
    Q = hip.DeviceBuffer(M * rb)
    tier_amd.rms_norm(X.ptr, t, K, R.ptr, K, f32(g).ptr, EPS, O.ptr if which == "h" else None, K,
                      O.ptr if which == "y" else None, K, Q.ptr if which == "q" else None, rb,
                      S.ptr if which == "q" else None, S.ptr if which == "rstd" else None, M, K)
    hip.synchronize()
    if which in "hy":
        assert np.array_equal(O.bits(), to_bits(t, h if which == "h" else y))
    elif which == "rstd":
        assert np.array_equal(S.download(np.float32), r)
    else:
        q, s = quantize(y)
        assert np.array_equal(Q.download(np.int8).reshape(M, rb)[:, :K], q) and np.array_equal(S.download(np.float32), s)


@pytest.mark.parametrize("K", [640, 5120, 40000])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_stream_updated_in_place(gpu, over, K):
    """h is x, or the residual: codes and h as with a buffer of its own."""
    M, t = 3, BF16
    xv, rv, g = rows(M, K, 7), rows(M, K, 8), gains(K)
    X, R = Rows(t, M, K, xv, 1), Rows(t, M, K, rv, 5)
    h, _, y = forward(t, X.values(), R.values(), g)
    H, rb, S = X if over == "x" else R, tier_amd.i8_row_bytes(K), f32(np.zeros(M))
    Q = hip.DeviceBuffer(M * rb)
    tier_amd.rms_norm(X.ptr, t, X.ld, R.ptr, R.ld, f32(g).ptr, EPS, H.ptr, H.ld, None, 0, Q.ptr, rb, S.ptr, None, M, K)
    hip.synchronize()
    q, s = quantize(y)
    assert np.array_equal(H.bits(), to_bits(t, h)) and H.outside_kept()
    assert np.array_equal(Q.download(np.int8).reshape(M, rb)[:, :K], q) and np.array_equal(S.download(np.float32), s)


def test_special_rows(gpu):
    """Zeros with and without eps, tiny and huge rows, NaN and infinities: as the formulas give them, and each row
    by itself."""
    K = 300
    x = rows(10, K, 9)
    x[0] = 0
    x[1] = 1e-30
    x[2] *= 1e30
    x[3, 5] = np.nan
    x[4, 299] = np.inf
    x[5, 0] = -np.inf
    x[6] = 2.0 ** -140
    x[7, 1:] = 0
    g = gains(K)
    for eps in (EPS, np.float32(0)):
        X, Y, S = Rows(F32, 10, K, x), Rows(F32, 10, K), f32(np.zeros(10))
        rb = tier_amd.i8_row_bytes(K)
        Q, M8 = hip.DeviceBuffer(10 * rb), MxRows(mx.E4M3, 10, K)
        tier_amd.rms_norm(X.ptr, F32, K, None, 0, f32(g).ptr, eps, None, 0, Y.ptr, K, Q.ptr, rb, S.ptr, None, 10, K)
        tier_amd.rms_norm_mx(X.ptr, F32, K, None, 0, f32(g).ptr, eps, None, 0, None, 0, mx.E4M3, M8.q.ptr, M8.rb, M8.s.ptr,
                             M8.sb, None, 10, K)
        hip.synchronize()
        _, _, y = forward(F32, x, None, g, eps)
        assert np.array_equal(Y.values().astype(np.float32), y, equal_nan=True)
        q, s = quantize(y)
        assert np.array_equal(Q.download(np.int8).reshape(10, rb)[:, :K], q)
        assert np.array_equal(S.download(np.float32), s, equal_nan=True)
        c, sc = M8.get()
        want, scales = mx.quantize(mx.E4M3, y)
        assert np.array_equal(sc, scales) and np.array_equal(c, want)


def test_codes_do_not_depend_on_the_launch(gpu):
    """The same row alone, among few and among many."""
    K, t = 5120, BF16
    x, g, rb = rows(600, K, 10), f32(gains(K)), tier_amd.i8_row_bytes(K)
    X, got = Rows(t, 600, K, x), []
    for M in (1, 8, 600):
        Q, S = hip.DeviceBuffer(M * rb), f32(np.zeros(M))
        tier_amd.rms_norm(X.ptr, t, K, None, 0, g.ptr, EPS, None, 0, None, 0, Q.ptr, rb, S.ptr, None, M, K)
        hip.synchronize()
        got.append((Q.download(np.int8)[:rb], S.download(np.float32)[0]))
    for q, s in got[1:]:
        assert np.array_equal(q, got[0][0]) and s == got[0][1]


@pytest.mark.parametrize("t,M,K", [(BF16, 4100, 4701), (F32, 2100, 4704), (F16, 700, 30000)])
def test_streamed_rows(gpu, t, M, K):
    """More bytes than the last-level cache keeps: rows past the caches, codes and sums as ever."""
    X, R, g, H = Rows(t, M, K, rows(M, K, 60)), Rows(t, M, K, rows(M, K, 61)), gains(K), Rows(t, M, K)
    h, r, y = forward(t, X.values(), R.values(), g)
    rb = tier_amd.i8_row_bytes(K)
    Q, S, RS = hip.DeviceBuffer(M * rb), f32(np.zeros(M)), f32(np.zeros(M))
    tier_amd.rms_norm(X.ptr, t, K, R.ptr, K, f32(g).ptr, EPS, H.ptr, K, None, 0, Q.ptr, rb, S.ptr, RS.ptr, M, K)
    hip.synchronize()
    q, s = quantize(y)
    assert np.array_equal(Q.download(np.int8).reshape(M, rb)[:, :K], q) and np.array_equal(S.download(np.float32), s)
    assert np.array_equal(H.bits(), to_bits(t, h)) and np.array_equal(RS.download(np.float32), r)
    DX, DG = Rows(t, M, K), f32(np.zeros(K))
    tier_amd.rms_norm_grad(X.ptr, t, K, H.ptr, K, f32(g).ptr, RS.ptr, R.ptr, K, DX.ptr, K, DG.ptr, M, K)
    hip.synchronize()
    check_grad(DX, DG.download(np.float32), X, H, R, r, g)


# -------------------------------------------------------------------- gradient
def check_grad(DX, got, DY, H, DH, r, g):
    """dx and dgain within the bound of the header comment."""
    M, K, t = H.rows, H.cols, H.t
    dhv, dyv, r64 = None if DH is None else DH.values(), DY.values(), r.astype(np.float64)
    want, dgain, xh, d, m = grad64(dyv, H.values(), r64, g.astype(np.float64), dhv)
    off = (64 + 6 + 16 + K / 1024) * U * np.abs(d * xh).mean(1, keepdims=True)
    err = 8 * U * (r64[:, None] * (np.abs(d) + np.abs(xh * m)) + (0 if dhv is None else np.abs(dhv))) + r64[:, None] * np.abs(xh) * off
    ok = np.abs(DX.values() - want) <= err + UNIT[t] * (np.abs(want) + err) + TINY[t]
    assert ok.all(), np.argwhere(~ok)[:5]
    assert (np.abs(got[:K] - dgain) <= (M + 64) * U * np.abs(dyv * xh).sum(0) + 1e-38).all()


def grad64(dy, h, r, g, dh):
    xh, d = h * r[:, None], dy * g
    m = (d * xh).mean(1, keepdims=True)
    dx = r[:, None] * (d - xh * m)
    return dx + (0 if dh is None else dh), (dy * xh).sum(0), xh, d, m


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,pad,skip", SIZES + [(1100, 640, 0, 0), (150, 17000, 1, 0), (390, 1000, 0, 2), (2100, 200, 0, 0)])
def test_gradient(gpu, t, M, K, pad, skip):
    H, DY, DH = Rows(t, M, K, rows(M, K, 11), pad, skip), Rows(t, M, K, rows(M, K, 12, 0.1), pad + 1), Rows(t, M, K, rows(M, K, 13, 0.1), 0, skip)
    g = gains(K)
    _, r, _ = forward(t, H.values(), None, g)
    n = tier_amd.rms_norm_grad_ws_bytes(M, K)
    for dh, own_ws in ((None, False), (DH, True)):
        DX, DG, ws = Rows(t, M, K, None, pad, skip), f32(np.full(K + 1, 5.0)), hip.DeviceBuffer(n + 16)
        ws.fill_bytes(0x55)
        tier_amd.rms_norm_grad(DY.ptr, t, DY.ld, H.ptr, H.ld, f32(g).ptr, f32(r).ptr, dh and dh.ptr, DH.ld, DX.ptr, DX.ld,
                               DG.ptr, M, K, ws.ptr if own_ws else None, n if own_ws else 0)
        hip.synchronize()
        got = DG.download(np.float32)
        check_grad(DX, got, DY, H, dh, r, g)
        assert got[K] == 5
        assert DX.outside_kept() and (ws.download(np.uint8)[n:] == 0x55).all()
        # without dgain: the same dx, no workspace
        D2 = Rows(t, M, K)
        tier_amd.rms_norm_grad(DY.ptr, t, DY.ld, H.ptr, H.ld, f32(g).ptr, f32(r).ptr, dh and dh.ptr, DH.ld, D2.ptr, K, None, M, K)
        hip.synchronize()
        assert np.array_equal(D2.bits(), DX.bits())


def test_gradient_against_differences():
    """The formula, in 64 bits, against central differences of the forward in 64 bits."""
    rng = np.random.default_rng(14)
    M, K, e = 3, 40, 1e-5
    x, dy, g = rng.standard_normal((M, K)), rng.standard_normal((M, K)), gains(K).astype(np.float64)

    def loss(x, g):
        return (dy * (x / np.sqrt((x ** 2).mean(1, keepdims=True) + EPS) * g)).sum()

    r = 1 / np.sqrt((x ** 2).mean(1) + EPS)
    dx, dgain, *_ = grad64(dy, x, r, g, None)
    for i, k in ((0, 0), (1, 17), (2, 39)):
        a, b = x.copy(), x.copy()
        a[i, k] += e
        b[i, k] -= e
        assert abs((loss(a, g) - loss(b, g)) / (2 * e) - dx[i, k]) < 1e-8
        ga, gb = g.copy(), g.copy()
        ga[k] += e
        gb[k] -= e
        assert abs((loss(x, ga) - loss(x, gb)) / (2 * e) - dgain[k]) < 1e-8


@pytest.mark.parametrize("K", [700, 40000])
@pytest.mark.parametrize("over", ["dy", "dh"])
def test_gradient_in_place(gpu, over, K):
    M, t = 5, F32
    H, g = Rows(t, M, K, rows(M, K, 15)), gains(K)
    _, r, _ = forward(t, H.values(), None, g)
    dyv, dhv, got = rows(M, K, 16), rows(M, K, 17), []
    for own in (True, False):
        DY, DH, DX = Rows(t, M, K, dyv, 2), Rows(t, M, K, dhv, 2), Rows(t, M, K, None, 2)
        to = DX if own else DY if over == "dy" else DH
        tier_amd.rms_norm_grad(DY.ptr, t, DY.ld, H.ptr, K, f32(g).ptr, f32(r).ptr, DH.ptr, DH.ld, to.ptr, to.ld, None, M, K)
        hip.synchronize()
        got.append(to.bits().copy())
    assert np.array_equal(*got)


def test_gradient_of_no_rows(gpu):
    DG = f32(np.full(9, 5.0))
    tier_amd.rms_norm_grad(None, F32, 8, None, 8, None, None, None, 0, None, 8, DG.ptr, 0, 8)
    hip.synchronize()
    assert DG.download(np.float32).tolist() == [0.0] * 8 + [5.0]


def test_captured(gpu):
    """Norm and gradient in one graph: every replay as the eager calls, on new rows."""
    M, K, t, st = 6, 1408, BF16, hip.Stream()
    g, X, R = f32(gains(K)), Rows(t, M, K, rows(M, K, 20)), Rows(t, M, K, rows(M, K, 21))
    rb, n = tier_amd.i8_row_bytes(K), tier_amd.rms_norm_grad_ws_bytes(M, K)

    def buffers():
        return (Rows(t, M, K), hip.DeviceBuffer(M * rb), hip.DeviceBuffer(M * 4), hip.DeviceBuffer(M * 4), Rows(t, M, K),
                hip.DeviceBuffer(K * 4), hip.DeviceBuffer(n))

    def call(b, s):
        H, Q, S, RS, DX, DG, ws = b
        tier_amd.rms_norm(X.ptr, t, K, R.ptr, K, g.ptr, EPS, H.ptr, K, None, 0, Q.ptr, rb, S.ptr, RS.ptr, M, K, s)
        tier_amd.rms_norm_grad(R.ptr, t, K, H.ptr, K, g.ptr, RS.ptr, X.ptr, K, DX.ptr, K, DG.ptr, M, K, ws.ptr, n, s)

    def all_bits(b):
        return [b[0].bits().copy(), b[1].download(np.uint8), b[2].download(np.uint8), b[3].download(np.uint8),
                b[4].bits().copy(), b[5].download(np.uint8)]

    mine, eager = buffers(), buffers()
    graph = hip.Graph(st, lambda s: call(mine, s))
    try:
        for i in range(3):
            hip.copy_d2d(X.ptr, Rows(t, M, K, rows(M, K, 30 + i)).ptr, M * K * 2)
            hip.synchronize()
            graph.launch(st)
            st.synchronize()
            call(eager, st)
            st.synchronize()
            for a, b in zip(all_bits(mine), all_bits(eager)):
                assert np.array_equal(a, b)
    finally:
        graph.destroy()
        st.destroy()
