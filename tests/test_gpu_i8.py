"""int8 products with a scale for each token and channel, against whole-number sums in numpy.

Codes and scales are exact by definition (three fp32 steps).  The sum is exact, so a result is off by
the rounding of the sum, of sx * sw, of their product, of the bias and of the output: 4 fp32 unit
roundoffs of |product| + |bias| and one of the output's type.
"""
import numpy as np
import pytest

import tier_amd
from rows import TINY, TYPES, UNIT, Rows, f32, i32
from tier_amd import hip

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def quantize(x):
    """(codes, scales) of fp32 rows by the definition in the header."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(1)
    q, s = np.zeros(x.shape, np.int64), np.full(len(x), np.nan, np.float32)
    for r in range(len(x)):
        if not np.isfinite(x[r]).all():
            continue
        m = top[r]
        pre = np.float32(2.0 ** 100) if m < np.float32(2.0 ** -100) else np.float32(1)
        s[r] = m / np.float32(127)
        if m > 0:
            inv = np.float32(127) / (m * pre)
            q[r] = np.rint((x[r] * pre) * inv).astype(np.int64)
    return q, s


def i8_rows(codes, rb=None, fill=0):
    """Device int8 rows of rb bytes: the codes, zeros to whole 128 bytes, `fill` behind."""
    rows, K = codes.shape
    need = tier_amd.i8_row_bytes(K)
    rb = need if rb is None else rb
    h = np.full((rows, rb), fill, np.int8)
    h[:, :need] = 0
    h[:, :K] = codes
    return hip.to_device(h), rb


def weight(N, K, seed, pad_fill=0):
    rng = np.random.default_rng(seed)
    w = np.clip(np.rint(rng.standard_normal((N, K)) * 40), -127, 127).astype(np.int64)
    rb = tier_amd.i8_row_bytes(K)
    h = np.full((N, rb), pad_fill, np.int8)
    h[:, :K] = w
    return w, (0.5 + rng.random(N)).astype(np.float32) * np.float32(0.02 / 40), hip.to_device(h), rb


def _x(M, K, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, ::53] *= 9
    return x


def check(got, t, q, sx, w, sw, bias=None):
    """got[m][n] against sx sw <q, w> + bias within the bound."""
    s = (q.astype(np.float64) @ w.T.astype(np.float64)) * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    b = np.zeros(s.shape[1]) if bias is None else bias.astype(np.float64)
    err = 4 * U * (np.abs(s) + np.abs(b))
    want = s + b
    dead = np.isnan(sx)
    assert np.isnan(got[dead]).all()
    ok = np.abs(got - want) <= err + UNIT[t] * (np.abs(want) + err) + TINY[t]
    assert ok[~dead].all(), np.argwhere(~ok & ~dead[:, None])[:5]


# ------------------------------------------------------------------- quantizer
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,pad,skip", [(1, 1, 0, 0), (3, 127, 0, 1), (2, 128, 3, 0), (5, 1408, 0, 0), (2, 5121, 2, 3),
                                          (3, 8192, 0, 0), (2, 16389, 0, 0), (1, 40000, 8, 8), (9, 2048, 0, 0),
                                          (2100, 130, 1, 0)])
def test_quant(gpu, t, M, K, pad, skip):
    x = _x(M, K, K + M)
    X = Rows(t, M, K, x, pad, skip)
    rb = tier_amd.i8_row_bytes(K) + (16 if pad else 0)
    Q, S = hip.DeviceBuffer(M * rb + 16), f32(np.full(M + 1, 7.0))
    Q.fill_bytes(0x55)
    tier_amd.i8_quant(X.ptr, t, X.ld, Q.ptr, rb, S.ptr, M, K)
    hip.synchronize()
    q, s = quantize(X.values())
    got = Q.download(np.int8)
    rows = got[:M * rb].reshape(M, rb)
    need = tier_amd.i8_row_bytes(K)
    assert np.array_equal(rows[:, :K], q) and not rows[:, K:need].any()
    assert (rows[:, need:] == 0x55).all() and (got[M * rb:] == 0x55).all()
    sc = S.download(np.float32)
    assert np.array_equal(sc[:M], s) and sc[M] == 7


def test_quant_special_rows(gpu):
    """Zeros, ties, one huge element, tiny and subnormal rows, NaN and infinities."""
    K = 300
    x = np.zeros((12, K), np.float32)
    x[1, :4] = [127, 0.5, 1.5, -2.5]           # ties go to the even code
    x[2, 7] = -3.0e38
    x[3] = 1e-3
    x[4, :3] = [2.0 ** -120, -2.0 ** -121, 2.0 ** -127]
    x[5, :2] = [1e-45, -1e-45]
    x[6, 299] = np.nan
    x[7, 0] = np.inf
    x[8, :2] = [np.inf, -np.inf]
    x[9] = -np.float32(2.0 ** -100)
    x[10] = np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    x[11] = np.float32(3.4028235e38)
    X, rb = Rows(tier_amd.F32, 12, K, x), tier_amd.i8_row_bytes(K)
    Q, S = hip.DeviceBuffer(12 * rb), f32(np.zeros(12))
    tier_amd.i8_quant(X.ptr, tier_amd.F32, K, Q.ptr, rb, S.ptr, 12, K)
    hip.synchronize()
    q, s = quantize(x)
    assert np.array_equal(Q.download(np.int8).reshape(12, rb)[:, :K], q)
    assert np.array_equal(S.download(np.float32), s, equal_nan=True)
    assert q[1, :4].tolist() == [127, 0, 2, -2] and s[0] == 0 and np.abs(q).max() == 127


# --------------------------------------------------------------------- product
SIZES = [(1, 1, 1), (1, 300, 515), (2, 129, 128), (3, 64, 1000), (4, 1030, 256), (5, 77, 640), (7, 513, 1408),
         (16, 200, 384), (17, 96, 2048), (33, 130, 129), (48, 1000, 512), (64, 257, 896), (65, 31, 300),
         (129, 260, 1030), (200, 640, 256), (300, 515, 200), (513, 770, 384)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_gemm(gpu, t, M, N, K):
    """Every size with a bias and odd strides; weights whose padding is not zero."""
    rng = np.random.default_rng(M + N + K)
    q = rng.integers(-127, 128, (M, K))
    sx = (0.5 + rng.random(M)).astype(np.float32)
    w, sw, W, rbw = weight(N, K, M + N, pad_fill=99)
    bias = rng.standard_normal(N).astype(np.float32) * 10
    X, rbx = i8_rows(q, tier_amd.i8_row_bytes(K) + 16, fill=77)
    Y = Rows(t, M, N, None, pad=N % 3, skip=N % 2)
    tier_amd.i8_gemm(X.ptr, rbx, f32(sx).ptr, W.ptr, rbw, f32(sw).ptr, f32(bias).ptr, Y.ptr, t, Y.ld, M, N, K)
    hip.synchronize()
    check(Y.values(), t, q, sx, w, sw, bias)
    assert Y.outside_kept()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_is_quant_and_gemm(gpu, t, M, N, K):
    """Within the bound of the codes' product, and bit for bit the two calls; both workspaces."""
    x = _x(M, K, K)
    w, sw, W, rbw = weight(N, K, 5)
    X, SW = Rows(t, M, K, x, pad=K % 4, skip=K % 2), f32(sw)
    q, sx = quantize(X.values())
    Y = Rows(t, M, N, None, pad=2)
    n = tier_amd.i8_linear_ws_bytes(M, N, K)
    ws = hip.DeviceBuffer(n)
    tier_amd.i8_linear(X.ptr, t, X.ld, W.ptr, rbw, SW.ptr, None, Y.ptr, t, Y.ld, M, N, K, ws.ptr, n)
    hip.synchronize()
    check(Y.values(), t, q, sx, w, sw)
    assert Y.outside_kept()
    rb = tier_amd.i8_row_bytes(K)
    Q, S, Y2, Y3 = hip.DeviceBuffer(M * rb), hip.DeviceBuffer(4 * M), Rows(t, M, N), Rows(t, M, N)
    tier_amd.i8_quant(X.ptr, t, X.ld, Q.ptr, rb, S.ptr, M, K)
    tier_amd.i8_gemm(Q.ptr, rb, S.ptr, W.ptr, rbw, SW.ptr, None, Y2.ptr, t, N, M, N, K)
    tier_amd.i8_linear(X.ptr, t, X.ld, W.ptr, rbw, SW.ptr, None, Y3.ptr, t, N, M, N, K)  # the library's pool
    hip.synchronize()
    assert np.array_equal(Y.bits(), Y2.bits()) and np.array_equal(Y.bits(), Y3.bits())


@pytest.mark.parametrize("M,N,K", [(1, 4096, 5120), (1, 1024, 14336), (4, 2816, 2048), (37, 5120, 1408), (1, 40, 40000),
                                   (3, 300, 66000), (1030, 2100, 640), (2049, 1030, 256)])
def test_larger_sizes(gpu, M, N, K):
    t = tier_amd.F32
    x = _x(M, K, 1)
    w, sw, W, rbw = weight(N, K, 2)
    X, Y = Rows(t, M, K, x), Rows(t, M, N)
    tier_amd.i8_linear(X.ptr, t, K, W.ptr, rbw, f32(sw).ptr, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    q, sx = quantize(x)
    check(Y.values(), t, q, sx, w, sw)


@pytest.mark.parametrize("M", [1, 3, 20, 140])
def test_largest_sums(gpu, M):
    """Codes of 127 all over, at the largest K: the sum stays below 2^31 (and -127 times 127 above -2^31)."""
    K, N, t = 133120, 3, tier_amd.F32
    w = np.full((N, K), 127, np.int64)
    w[1] = -127
    W, rbw = i8_rows(w)
    q = np.full((M, K), 127, np.int64)
    X, rbx = i8_rows(q)
    one, Y = np.ones(M, np.float32), Rows(t, M, N)
    tier_amd.i8_gemm(X.ptr, rbx, f32(one).ptr, W.ptr, rbw, f32(np.ones(N)).ptr, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    check(Y.values(), t, q, one, w, np.ones(N, np.float32))
    x = Rows(t, M, K, np.full((M, K), 2.0))
    tier_amd.i8_linear(x.ptr, t, K, W.ptr, rbw, f32(np.ones(N)).ptr, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    check(Y.values(), t, q, np.full(M, np.float32(2) / np.float32(127)), w, np.ones(N, np.float32))


@pytest.mark.parametrize("M", [1, 4, 30, 150])
def test_nonfinite_and_zero_rows(gpu, M):
    """A NaN or an infinity makes its own row NaN and no other; a zero row gives the bias."""
    t, N, K = tier_amd.F32, 200, 700
    for r, bad in ((0, np.nan), (M - 1, np.inf), (M // 2, -np.inf), (0, 0.0)):
        x = _x(M, K, 3)
        if bad == 0.0:
            x[r] = 0
        else:
            x[r, K - 1] = bad
        w, sw, W, rbw = weight(N, K, 4)
        bias = np.linspace(-1, 1, N).astype(np.float32)
        X, Y = Rows(t, M, K, x), Rows(t, M, N)
        tier_amd.i8_linear(X.ptr, t, K, W.ptr, rbw, f32(sw).ptr, f32(bias).ptr, Y.ptr, t, N, M, N, K)
        hip.synchronize()
        q, sx = quantize(x)
        check(Y.values(), t, q, sx, w, sw, bias)
        if bad == 0.0:
            assert np.array_equal(Y.values()[r], bias.astype(np.float64))


def test_input_gradient(gpu):
    """dX = dY W as the product of dY's codes with W transposed and quantized by its own rows: within
    the two quantizers' half steps of the formula, and so of differences of <dY, x W^T>."""
    t, M, N, K = tier_amd.F32, 40, 384, 260
    rng = np.random.default_rng(6)
    w = (rng.standard_normal((N, K)) * 0.02).astype(np.float32)
    dy = rng.standard_normal((M, N)).astype(np.float32)
    rb = tier_amd.i8_row_bytes(N)
    WT, Q, S = Rows(t, K, N, w.T), hip.DeviceBuffer(K * rb), hip.DeviceBuffer(4 * K)
    tier_amd.i8_quant(WT.ptr, t, N, Q.ptr, rb, S.ptr, K, N)
    DY, DX = Rows(t, M, N, dy), Rows(t, M, K)
    tier_amd.i8_linear(DY.ptr, t, N, Q.ptr, rb, S.ptr, None, DX.ptr, t, K, M, K, N)
    hip.synchronize()
    got = DX.values()
    q, sd = quantize(dy)
    wq, sw = quantize(w.T)
    check(got, t, q, sd, wq, sw)
    half_d, half_w = 0.501 * sd.astype(np.float64), 0.501 * sw.astype(np.float64)
    a, b = np.abs(dy).astype(np.float64), np.abs(w.T).astype(np.float64)
    bound = half_d[:, None] * b.sum(1) + a.sum(1)[:, None] * half_w + N * half_d[:, None] * half_w
    assert np.all(np.abs(got - dy.astype(np.float64) @ w) <= bound)
    v, h, w64 = rng.standard_normal((M, K)), 0.5, w.astype(np.float64)
    L = lambda x: (dy * (x @ w64.T)).sum()  # noqa: E731
    assert abs((L(h * v) - L(-h * v)) / (2 * h) - (got * v).sum()) <= (bound * np.abs(v)).sum()


# --------------------------------------------------------------------- experts
def _routed(T, k, E, seed, drop=0.2):
    rng = np.random.default_rng(seed)
    ids = np.argsort(rng.random((T, max(E, k))), 1)[:, :k].astype(np.int32) % E
    ids[rng.random((T, k)) < drop] = -1
    return ids


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 5, 3), (1, 8, 64, 96, 256), (8, 8, 64, 130, 200), (30, 2, 3, 257, 384),
                                       (100, 4, 5, 64, 1408), (90, 6, 130, 33, 128), (300, 2, 2, 300, 130),
                                       (700, 3, 6, 520, 256)])
def test_grouped(gpu, t, T, k, E, N, K):
    """Gathered through the plan, with dropped pairs, empty experts and ragged counts."""
    ids = _routed(T, k, E, T + N)
    P = T * k
    x = _x(T, K, 9)
    w, sw, W, rbw = weight(E * N, K, 10, pad_fill=55)
    X, rb = Rows(t, T, K, x), tier_amd.i8_row_bytes(K)
    Q, S, Y = hip.DeviceBuffer(T * rb), hip.DeviceBuffer(4 * T), Rows(t, P, N, None, pad=N % 2, skip=N % 3)
    OF, TP, SP = i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P))
    tier_amd.moe_plan(i32(ids).ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr)
    tier_amd.i8_quant(X.ptr, t, K, Q.ptr, rb, S.ptr, T, K)
    tier_amd.i8_gemm_grouped(Q.ptr, rb, S.ptr, SP.ptr, T, k, OF.ptr, E, W.ptr, rbw, f32(sw).ptr, Y.ptr, t, Y.ld, P, N, K)
    hip.synchronize()
    off, srt = OF.download(np.int32), SP.download(np.int32)
    q, sx = quantize(X.values())
    y = Y.values()
    for e in range(E):
        r = srt[off[e]:off[e + 1]] // k
        check(y[off[e]:off[e + 1]], t, q[r], sx[r], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])
    assert not y[off[E]:].any() and Y.outside_kept()


def test_grouped_rows_in_place(gpu):
    """No row index: row p of Y is row p of x; rows past x and past the experts are zeros."""
    t, E, N, K, P = tier_amd.F32, 4, 70, 300, 60
    rng = np.random.default_rng(3)
    off = np.array([0, 11, 11, 47, 55], np.int32)
    q = rng.integers(-127, 128, (50, K))
    X, rb = i8_rows(q)
    sx = np.ones(50, np.float32)
    w, sw, W, rbw = weight(E * N, K, 1)
    Y = Rows(t, P, N)
    tier_amd.i8_gemm_grouped(X.ptr, rb, f32(sx).ptr, None, 50, 1, i32(off).ptr, E, W.ptr, rbw, f32(sw).ptr, Y.ptr, t, N,
                             P, N, K)
    hip.synchronize()
    y = Y.values()
    for e in range(E):
        b = min(off[e + 1], 50)
        check(y[off[e]:b], t, q[off[e]:b], sx[off[e]:b], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])
    assert not y[50:].any()


def test_grouped_many_rows(gpu):
    """Experts with hundreds of rows: one full, one empty, one of one row, ragged rest."""
    t, T, k, E, N, K = tier_amd.BF16, 2300, 2, 7, 640, 512
    rng = np.random.default_rng(12)
    ids = rng.choice(E, size=(T, k), p=[0.4, 0, 0.25, 0.15, 0.1, 0.1, 0]).astype(np.int32)
    ids[5, 0] = 6
    x, P = _x(T, K, 2), T * k
    w, sw, W, rbw = weight(E * N, K, 7)
    X, rb = Rows(t, T, K, x), tier_amd.i8_row_bytes(K)
    Q, S, Y = hip.DeviceBuffer(T * rb), hip.DeviceBuffer(4 * T), Rows(t, P, N)
    OF, TP, SP = i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P))
    tier_amd.moe_plan(i32(ids).ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr)
    tier_amd.i8_quant(X.ptr, t, K, Q.ptr, rb, S.ptr, T, K)
    tier_amd.i8_gemm_grouped(Q.ptr, rb, S.ptr, SP.ptr, T, k, OF.ptr, E, W.ptr, rbw, f32(sw).ptr, Y.ptr, t, N, P, N, K)
    hip.synchronize()
    off, srt, y = OF.download(np.int32), SP.download(np.int32), Y.values()
    q, sx = quantize(X.values())
    for e in range(E):
        r = srt[off[e]:off[e + 1]] // k
        check(y[off[e]:off[e + 1]], t, q[r], sx[r], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,k,E,N,K", [(200, 1, 9, 1010, 130), (500, 1, 9, 3500, 130), (3000, 3, 33, 300, 512),
                                       (500, 1, 9, 5000, 130), (3000, 3, 33, 1010, 130), (2000, 1, 33, 2050, 130),
                                       (1100, 2, 3, 1000, 260)])
def test_grouped_tiles(gpu, t, T, k, E, N, K):
    """The tiles of 64 to 256 rows, with 20 to 700 rows an expert: wholly, by half of a wave's blocks, by none of them."""
    ids, P = _routed(T, k, E, T + N, drop=0.1), T * k
    q = np.random.default_rng(N).integers(-127, 128, (T, K))
    X, rb = i8_rows(q)
    sx = np.random.default_rng(T).random(T).astype(np.float32)
    w, sw, W, rbw = weight(E * N, K, 13)
    OF, TP, SP, Y = i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P)), Rows(t, P, N)
    tier_amd.moe_plan(i32(ids).ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr)
    tier_amd.i8_gemm_grouped(X.ptr, rb, f32(sx).ptr, SP.ptr, T, k, OF.ptr, E, W.ptr, rbw, f32(sw).ptr, Y.ptr, t, N, P, N, K)
    hip.synchronize()
    off, srt, y = OF.download(np.int32), SP.download(np.int32), Y.values()
    for e in range(E):
        r = srt[off[e]:off[e + 1]] // k
        check(y[off[e]:off[e + 1]], t, q[r], sx[r], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])
    assert not y[off[E]:].any()


@pytest.mark.parametrize("M", [1, 6, 50, 300])
def test_in_a_graph(gpu, M):
    """A captured linear on a stream of its own replays on new inputs as the eager call."""
    t, N, K = tier_amd.F32, 520, 640
    w, sw, W, rbw = weight(N, K, 11)
    X, Y, SW = Rows(t, M, K, _x(M, K, 0)), Rows(t, M, N), f32(sw)
    n = tier_amd.i8_linear_ws_bytes(M, N, K)
    ws, s = hip.DeviceBuffer(n), hip.Stream()
    call = lambda st: tier_amd.i8_linear(X.ptr, t, K, W.ptr, rbw, SW.ptr, None, Y.ptr, t, N, M, N, K, ws.ptr, n,  # noqa: E731
                                         stream=st)
    g = hip.Graph(s, call)
    for seed in (21, 22, 23):
        x = _x(M, K, seed)
        X.buf.upload(x)
        hip.synchronize()
        g.launch(s)
        s.synchronize()
        replayed = Y.bits().copy()
        q, sx = quantize(x)
        check(Y.values(), t, q, sx, w, sw)
        call(s)
        s.synchronize()
        assert np.array_equal(Y.bits(), replayed)
    g.destroy()
    s.destroy()


@pytest.mark.parametrize("M", [1, 2, 10, 140])
def test_offsets_past_32_bits(gpu, M):
    """Rows of W, x and Y 32 MiB apart: the last ones start past 4 GiB."""
    t, N, K, far = tier_amd.F32, 140, 100, 1 << 25
    rng = np.random.default_rng(M)
    w, sw, _, _ = weight(N, K, 1)
    W = hip.DeviceBuffer((N - 1) * far + 128)
    for n in range(N):
        W.upload(np.pad(w[n], (0, 28)).astype(np.int8), n * far)
    x = _x(M, K, 8)
    X, Y = hip.DeviceBuffer((M - 1) * far + 4 * K), hip.DeviceBuffer((M - 1) * far + 4 * N)
    for m in range(M):
        X.upload(x[m], m * far)
    tier_amd.i8_linear(X.ptr, t, far // 4, W.ptr, far, f32(sw).ptr, None, Y.ptr, t, far // 4, M, N, K)
    hip.synchronize()
    q, sx = quantize(x)
    check(np.stack([Y.download(np.float32, N, m * far) for m in range(M)]).astype(np.float64), t, q, sx, w, sw)


def test_experts_past_32_bits(gpu):
    """Experts' weights 2.3 GB apart, gathered by rows in any order (one of them pointing nowhere)."""
    t, E, N, K, far = tier_amd.BF16, 3, 70, 128, 1 << 25
    w, sw, _, _ = weight(E * N, K, 2)
    W = hip.DeviceBuffer((E * N - 1) * far + 128)
    for n in range(E * N):
        W.upload(w[n].astype(np.int8), n * far)
    q = np.random.default_rng(3).integers(-127, 128, (6, K))
    X, rb = i8_rows(q)
    sx, rows = np.ones(6, np.float32), np.array([5, 0, 3, 99, 1, 2, 4, 0, 5], np.int32)
    off, Y = np.array([0, 2, 4, 9], np.int32), Rows(t, 9, N)
    tier_amd.i8_gemm_grouped(X.ptr, rb, f32(sx).ptr, i32(rows).ptr, 6, 1, i32(off).ptr, E, W.ptr, far, f32(sw).ptr, Y.ptr, t,
                             N, 9, N, K)
    hip.synchronize()
    y = Y.values()
    assert not y[3].any()
    for e in range(E):
        for p in range(off[e], off[e + 1]):
            if p != 3:
                check(y[p:p + 1], t, q[rows[p]][None], sx[:1], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])


def test_every_tile(gpu):
    """Sizes at which each tile of the cost table is the least dear, with ragged rows and columns."""
    t = tier_amd.BF16
    for M, N, K in ((6, 1003, 640), (6, 1003, 260), (6, 10001, 260), (50, 2501, 260), (50, 5101, 2600), (50, 5101, 640),
                    (50, 5101, 260), (30, 20001, 260), (130, 20001, 1300), (401, 20001, 260), (401, 28001, 640),
                    (2051, 8001, 260)):
        rng = np.random.default_rng(M)
        q = rng.integers(-127, 128, (M, K))
        sx = (0.5 + rng.random(M)).astype(np.float32)
        w, sw, W, rbw = weight(N, K, N, pad_fill=-3)
        X, rbx = i8_rows(q)
        Y = Rows(t, M, N, None, pad=1)
        tier_amd.i8_gemm(X.ptr, rbx, f32(sx).ptr, W.ptr, rbw, f32(sw).ptr, None, Y.ptr, t, Y.ld, M, N, K)
        hip.synchronize()
        rows = np.unique(np.concatenate([rng.choice(M, min(M, 60), replace=False), [0, M - 1]]))
        check(Y.values()[rows], t, q[rows], sx[rows], w, sw)
        assert Y.outside_kept(), (M, N, K)
