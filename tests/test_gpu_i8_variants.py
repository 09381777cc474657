"""The kernel variants that sizes choose between, each in every row type: the GEMV of two rows of W a wave,
the quantizer's forms, every tile with a bias, long plans, and the routed product in a captured graph.
Bounds as in test_gpu_i8.py and test_gpu_moe_rows.py."""
import numpy as np
import pytest

import tier_amd
from rows import SIZE, TYPES, Rows, f32, i32
from test_gpu_i8 import _routed, _x, check, i8_rows, quantize, weight
from tier_amd import hip

pytestmark = pytest.mark.gpu


# N from 5120 up: 16 waves of two rows each
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [1, 2])
@pytest.mark.parametrize("N,K,bias", [(5120, 640, True), (5121, 1030, True), (5151, 200, False), (7001, 2100, True)])
def test_linear_two_rows_a_wave(gpu, t, M, N, K, bias):
    w, sw, W, rbw = weight(N, K, N, pad_fill=11)
    X, Y = Rows(t, M, K, _x(M, K, M), pad=1, skip=K % 2), Rows(t, M, N, None, pad=3, skip=1)
    b = np.random.default_rng(N).standard_normal(N).astype(np.float32) if bias else None
    SW, B = f32(sw), f32(b) if bias else None
    tier_amd.i8_linear(X.ptr, t, X.ld, W.ptr, rbw, SW.ptr, B.ptr if bias else None, Y.ptr, t, Y.ld, M, N, K)
    hip.synchronize()
    q, sx = quantize(X.values())
    check(Y.values(), t, q, sx, w, sw, b)
    assert Y.outside_kept()
    Q, rb = i8_rows(q)
    Z = Rows(t, M, N)
    tier_amd.i8_gemm(Q.ptr, rb, f32(sx).ptr, W.ptr, rbw, SW.ptr, B.ptr if bias else None, Z.ptr, t, N, M, N, K)
    hip.synchronize()
    assert np.array_equal(Y.bits(), Z.bits())


# units of 16 bytes a row: each number of registers, 256 and 1024 threads, and rows read twice
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,units", [(520, 300), (520, 700), (520, 1500), (515, 3000), (513, 4200), (3, 900), (3, 1500),
                                     (3, 3000), (3, 4200)])
def test_quantizer_forms(gpu, t, M, units):
    K = units * 16 // SIZE[t] - 3
    x = _x(M, K, units)
    x[1] = 0
    x[2, K - 1] = 1000
    X, rb = Rows(t, M, K, x, pad=1), tier_amd.i8_row_bytes(K)
    Q, S = hip.DeviceBuffer(M * rb + 64), f32(np.full(M + 1, 7.0))
    Q.fill_bytes(0x55)
    tier_amd.i8_quant(X.ptr, t, X.ld, Q.ptr, rb, S.ptr, M, K)
    hip.synchronize()
    q, s = quantize(X.values())
    got = Q.download(np.int8)
    rows = got[:M * rb].reshape(M, rb)
    assert np.array_equal(rows[:, :K], q) and not rows[:, K:].any() and (got[M * rb:] == 0x55).all()
    assert np.array_equal(S.download(np.float32), np.append(s, np.float32(7)))


# sizes at which each dense tile is the least dear
TILES = [(6, 1003, 640), (6, 1003, 260), (6, 10001, 260), (50, 2501, 260), (50, 5101, 2600), (50, 5101, 640),
         (50, 5101, 260), (30, 20001, 260), (130, 20001, 1300), (401, 20001, 260), (401, 28001, 640), (2051, 8001, 260)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", TILES)
def test_every_tile_with_a_bias(gpu, t, M, N, K):
    rng = np.random.default_rng(M)
    q = rng.integers(-127, 128, (M, K))
    sx = ((0.5 + rng.random(M)) * 0.1).astype(np.float32)
    w, sw, W, rbw = weight(N, K, N)
    bias = (10 * rng.standard_normal(N)).astype(np.float32)
    X, rbx = i8_rows(q)
    Y = Rows(t, M, N, None, pad=N % 2, skip=1)
    tier_amd.i8_gemm(X.ptr, rbx, f32(sx).ptr, W.ptr, rbw, f32(sw).ptr, f32(bias).ptr, Y.ptr, t, Y.ld, M, N, K)
    hip.synchronize()
    rows = np.unique(np.concatenate([rng.choice(M, min(M, 40), replace=False), [0, M - 1]]))
    check(Y.values()[rows], t, q[rows], sx[rows], w, sw, bias)
    assert Y.outside_kept()


def _plan(ids, E):
    """offsets, places, sorted pairs by definition."""
    flat = ids.ravel()
    key = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(key, kind="stable").astype(np.int32)
    off = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1))]).astype(np.int32)
    srt = order.copy()
    srt[off[E]:] = -1
    places = np.full(flat.size, -1, np.int32)
    places[order[:off[E]]] = np.arange(off[E])
    return off[:E + 1], places, srt


# 1024 pairs a chunk up to 262144 of them, 4096 above (the last chunk ragged); the largest plan
@pytest.mark.parametrize("T,k,E,drop", [(65536, 4, 64, 0.1), (65537, 4, 64, 0.1), (37501, 8, 1024, 0.0), (300007, 1, 1, 0.5),
                                        (1 << 20, 8, 1024, 0.05)])
def test_long_plans(gpu, T, k, E, drop):
    rng = np.random.default_rng(E)
    ids = np.minimum(rng.integers(0, E + E // 4 + 1, (T, k)), E - 1).astype(np.int32)  # the last expert fuller
    ids[rng.random((T, k)) < drop] = -1
    P, n = T * k, tier_amd.moe_plan_ws_bytes(T, k, E)
    O, TP, SP, ws = i32(np.full(E + 2, 77)), i32(np.full(P + 1, 77)), i32(np.full(P + 1, 77)), hip.DeviceBuffer(n + 64)
    ws.fill_bytes(0x55)
    tier_amd.moe_plan(i32(ids).ptr, T, k, E, O.ptr, TP.ptr, SP.ptr, ws.ptr, n)
    hip.synchronize()
    off, places, srt = _plan(ids, E)
    assert np.array_equal(O.download(np.int32), np.append(off, 77))
    assert np.array_equal(TP.download(np.int32), np.append(places, 77))
    assert np.array_equal(SP.download(np.int32), np.append(srt, 77))
    assert (ws.download(np.uint8)[n:] == 0x55).all()


# tiles of 16, 64 and 256 rows; one and two launches of the plan
@pytest.mark.parametrize("T,k,E,N,K", [(8, 4, 12, 130, 256), (200, 1, 9, 1010, 130), (2200, 2, 3, 1000, 260),
                                       (8300, 4, 40, 72, 128)])
def test_routed_product_in_a_graph(gpu, T, k, E, N, K):
    """Plan, quantizer, gathered product and weighted sum captured once: replays follow new routings, with
    eager work between them, and give the eager calls' bits."""
    t, P, rng = tier_amd.F32, T * k, np.random.default_rng(T)
    w, sw, W, rbw = weight(E * N, K, 3)
    rb, n, x = tier_amd.i8_row_bytes(K), tier_amd.moe_plan_ws_bytes(T, k, E), _x(T, K, 9)
    wt = rng.random((T, k)).astype(np.float32)
    D, OF, TP, SP = i32(_routed(T, k, E, 0)), i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P))
    X, Y, O, SW, WT = Rows(t, T, K, x), Rows(t, P, N), Rows(t, T, N), f32(sw), f32(wt)
    Q, S, ws = hip.DeviceBuffer(T * rb), hip.DeviceBuffer(4 * T), hip.DeviceBuffer(max(n, 4))

    def step(s):
        tier_amd.moe_plan(D.ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr, ws.ptr, n, stream=s)
        tier_amd.i8_quant(X.ptr, t, K, Q.ptr, rb, S.ptr, T, K, stream=s)
        tier_amd.i8_gemm_grouped(Q.ptr, rb, S.ptr, SP.ptr, T, k, OF.ptr, E, W.ptr, rbw, SW.ptr, Y.ptr, t, N, P, N, K,
                                 stream=s)
        tier_amd.moe_unsort(Y.ptr, t, N, TP.ptr, WT.ptr, O.ptr, N, T, k, N, stream=s)

    s = hip.Stream()
    g = hip.Graph(s, step)
    q, sx = quantize(x)
    for seed in (1, 2, 3):
        ids = _routed(T, k, E, seed, drop=0.2 * (seed - 1))
        D.upload(ids)
        hip.synchronize()
        g.launch(s)
        s.synchronize()
        off, places, srt = _plan(ids, E)
        assert np.array_equal(OF.download(np.int32), off) and np.array_equal(SP.download(np.int32), srt)
        y, bits, out = Y.values(), Y.bits().copy(), O.bits().copy()
        for e in range(E):
            r = srt[off[e]:off[e + 1]] // k
            check(y[off[e]:off[e + 1]], t, q[r], sx[r], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])
        assert not y[off[E]:].any()
        at = places.reshape(T, k)
        terms = np.where(at[..., None] >= 0, y[np.maximum(at, 0)] * wt.astype(np.float64)[..., None], 0.0)
        assert np.all(np.abs(O.values() - terms.sum(1)) <= (k + 1) * 2.0 ** -24 * np.abs(terms).sum(1))
        step(s)
        s.synchronize()
        assert np.array_equal(Y.bits(), bits) and np.array_equal(O.bits(), out)
    g.destroy()
    s.destroy()
