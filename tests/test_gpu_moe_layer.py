"""A routed int8 layer of a few tokens, against its definition.

Sums of codes are whole numbers, gate and up two fp32 roundings of them, h one rounding of a 64-bit value: the
codes of h are fixed by these steps and made the same way here.  An output is then off by the roundings of each
pair's product (4 fp32 unit roundoffs of it), of its weighting and addition (one each of the sums of magnitudes,
for each pair), and of the output's type.
"""
import numpy as np
import pytest

import tier_amd
from rows import TINY, TYPES, UNIT, Rows, f32, i32
from test_gpu_i8 import i8_rows, quantize
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, F16, BF16 = tier_amd.F32, tier_amd.F16, tier_amd.BF16
U = 2.0 ** -24


class Experts:
    """E int8 experts on the device and on the host."""

    def __init__(self, E, K, F, seed, pad=0):
        rng = np.random.default_rng(seed)
        self.E, self.K, self.F = E, K, F
        self.gu = np.clip(np.rint(rng.standard_normal((E * 2 * F, K)) * 40), -127, 127).astype(np.int64)
        self.d = np.clip(np.rint(rng.standard_normal((E * K, F)) * 40), -127, 127).astype(np.int64)
        self.sg = ((0.5 + rng.random(E * 2 * F)) * 0.02 / 40).astype(np.float32)
        self.sd = ((0.5 + rng.random(E * K)) * 0.02 / 40).astype(np.float32)
        self.G, self.rbg = i8_rows(self.gu, tier_amd.i8_row_bytes(K) + pad, 0x55)
        self.D, self.rbd = i8_rows(self.d, tier_amd.i8_row_bytes(F) + 2 * pad, 0x55)
        self.SG, self.SD = f32(self.sg), f32(self.sd)


def layer(ex, q, sx, ids, w):
    """(out, sum of magnitudes) in 64 bits behind the codes of h."""
    T, k = ids.shape
    E, K, F = ex.E, ex.K, ex.F
    out, mag = np.zeros((T, K)), np.zeros((T, K))
    with np.errstate(all="ignore"):
        for t in range(T):
            for j in range(k):
                e = ids[t, j]
                if not 0 <= e < E:
                    continue
                ch = slice(2 * F * e, 2 * F * (e + 1))
                s = (ex.gu[ch] @ q[t]).astype(np.float32) * (sx[t] * ex.sg[ch])
                g, u = s[:F].astype(np.float64), s[F:].astype(np.float64)
                h = (g / (1 + np.exp(-g)) * u).astype(np.float32)
                hq, sh = quantize(h[None])
                ch = slice(K * e, K * (e + 1))
                y = (ex.d[ch] @ hq[0]).astype(np.float64) * sh[0].astype(np.float64) * ex.sd[ch].astype(np.float64)
                out[t] += float(w[t, j]) * y
                mag[t] += np.abs(float(w[t, j]) * y)
    return out, mag


def run(ex, q, sx, ids, w, t=F32, pad=0, ws=None, n=0, stream=None, X=None):
    T, k = ids.shape
    Xq, rb = i8_rows(q) if X is None else X
    Y = Rows(t, T, ex.K, None, pad, pad and 1)
    tier_amd.moe_i8_layer(Xq.ptr, rb, f32(sx).ptr, i32(ids).ptr, f32(w).ptr, ex.G.ptr, ex.rbg, ex.SG.ptr, ex.D.ptr, ex.rbd,
                          ex.SD.ptr, Y.ptr, t, Y.ld, T, k, ex.E, ex.K, ex.F, ws, n, stream)
    hip.synchronize()
    assert Y.outside_kept()
    return Y


def check(Y, ex, q, sx, ids, w):
    want, mag = layer(ex, q, sx, ids, w)
    got, t = Y.values(), Y.t
    err = (4 + 2 * ids.shape[1]) * U * mag
    dead = np.isnan(want)
    assert np.isnan(got[dead]).all()
    ok = np.abs(got - want) <= err + UNIT[t] * (np.abs(want) + err) + TINY[t]
    assert ok[~dead].all(), (np.argwhere(~ok & ~dead)[:5], np.nanmax(np.abs(got - want)))


def tokens(T, K, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, K)).astype(np.float32)
    x[:, ::53] *= 6
    return quantize(x)


def routes(T, k, E, seed):
    rng = np.random.default_rng(seed)
    ids = np.argsort(rng.random((T, E)), 1)[:, :k].astype(np.int32)
    w = rng.random((T, k)).astype(np.float32)
    return ids, w / w.sum(1, keepdims=True)


SHAPES = [(1, 1, 1, 1, 1), (1, 2, 4, 130, 33), (1, 8, 64, 512, 704), (2, 3, 5, 1000, 100), (5, 2, 8, 384, 1408),
          (8, 8, 16, 256, 96), (16, 1, 3, 640, 257), (17, 4, 4, 200, 48), (33, 2, 6, 96, 300), (64, 8, 16, 160, 64),
          (3, 1, 1024, 16, 16), (64, 6, 40, 64, 80), (1, 8, 8, 2048, 1408), (4, 2, 2, 48, 4200), (1, 32, 40, 64, 32)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,k,E,K,F", SHAPES)
def test_layer(gpu, t, T, k, E, K, F):
    pad = 16 if T % 2 else 0
    ex = Experts(E, K, F, K + F, pad)
    q, sx = tokens(T, K, T)
    ids, w = routes(T, k, E, T + k)
    check(run(ex, q, sx, ids, w, t, pad=T % 3), ex, q, sx, ids, w)


def test_dropped_and_repeated(gpu):
    """Ids outside the experts, whatever stands in their weights; a token of none; an expert twice for one token; all
    pairs on one expert."""
    E, K, F = 6, 300, 150
    ex = Experts(E, K, F, 1)
    q, sx = tokens(9, K, 2)
    ids, w = routes(9, 4, E, 3)
    ids[0] = -1
    ids[1, 2], ids[2, 0], ids[3, 3] = E, np.iinfo(np.int32).max, np.iinfo(np.int32).min
    w[0], w[1, 2], w[2, 0], w[3, 3] = np.nan, np.nan, np.inf, np.nan
    ids[4] = 2
    ids[5, 1] = ids[5, 3]
    Y = run(ex, q, sx, ids, w)
    check(Y, ex, q, sx, ids, w)
    assert not Y.values()[0].any()
    ids[:] = -7
    assert not run(ex, q, sx, ids, w, BF16).values().any()
    ids[:] = 5
    w[:] = 0.25
    check(run(ex, q, sx, ids, w), ex, q, sx, ids, w)


@pytest.mark.parametrize("E", [2, 600])
def test_most_pairs_on_one_expert(gpu, E):
    """64 tokens, all 512 pairs on one expert, and beside it single ones."""
    K, F = 64, 48
    ex = Experts(E, K, F, 4)
    q, sx = tokens(64, K, 5)
    rng = np.random.default_rng(6)
    ids, w = np.full((64, 8), 1, np.int32), rng.random((64, 8)).astype(np.float32)
    check(run(ex, q, sx, ids, w, F16), ex, q, sx, ids, w)
    ids[7, 3] = 0
    check(run(ex, q, sx, ids, w), ex, q, sx, ids, w)


def test_far_rows(gpu):
    """A NaN token, a zero token, far scales, an activation that saturates: each token by itself."""
    E, K, F = 4, 200, 90
    ex = Experts(E, K, F, 7)
    q, sx = tokens(8, K, 8)
    ids, w = routes(8, 2, E, 9)
    q[1], sx[1] = 0, np.nan
    q[2], sx[2] = 0, 0
    sx[3], sx[4], sx[5] = 1e4, 1e-30, 3e-38
    Y = run(ex, q, sx, ids, w)
    check(Y, ex, q, sx, ids, w)
    assert np.isnan(Y.values()[1]).all() and not Y.values()[2].any()
    alone = [run(ex, q[i:i + 1], sx[i:i + 1], ids[i:i + 1], w[i:i + 1]).bits() for i in range(8)]
    assert np.array_equal(np.concatenate(alone), Y.bits())  # no token depends on the others, bit for bit


def test_results_do_not_depend_on_the_call(gpu):
    """64 tokens at once, and the same in calls of 1, 5 and 33: bit for bit."""
    E, K, F, k = 9, 260, 200, 4
    ex = Experts(E, K, F, 70)
    q, sx = tokens(64, K, 71)
    ids, w = routes(64, k, E, 72)
    whole = run(ex, q, sx, ids, w).bits()
    for n in (1, 5, 33):
        parts = [run(ex, q[i:i + n], sx[i:i + n], ids[i:i + n], w[i:i + n]).bits() for i in range(0, 64, n)]
        assert np.array_equal(np.concatenate(parts), whole), n


def test_every_code(gpu):
    """Codes of -127 and 127 everywhere: the largest sums."""
    E, K, F = 2, 1024, 640
    ex = Experts(E, K, F, 10)
    ex.gu[:] = np.where(ex.gu > 0, 127, -127)
    ex.d[:] = np.where(ex.d > 0, 127, -127)
    ex.gu[0] = ex.d[0] = 127
    (ex.G, ex.rbg), (ex.D, ex.rbd) = i8_rows(ex.gu), i8_rows(ex.d)
    q, sx = tokens(3, K, 11)
    q[:] = np.where(q > 0, 127, -127)
    q[0] = 127
    ids, w = routes(3, 2, E, 12)
    check(run(ex, q, sx, ids, w), ex, q, sx, ids, w)


@pytest.mark.parametrize("T,k,E", [(1, 2, 8), (7, 3, 5), (16, 4, 6), (2, 2, 40)])
def test_captured_follows_the_routing(gpu, T, k, E):
    """Replays of one graph on new routings and rows, its own workspace, eager calls of another between them."""
    K, F, st = 256, 130, hip.Stream()
    ex = Experts(E, K, F, 13)
    X, rb = i8_rows(np.zeros((T, K), np.int64))
    S, I, W, Y = hip.DeviceBuffer(T * 4), hip.DeviceBuffer(T * k * 4), hip.DeviceBuffer(T * k * 4), Rows(BF16, T, K)
    n = tier_amd.moe_i8_layer_ws_bytes(T, k, K, F)
    ws, ws2 = hip.DeviceBuffer(n + 16), hip.DeviceBuffer(n + 16)
    ws.fill_bytes(0x55)
    ws2.fill_bytes(0xff)

    def call(y, w_s, s):
        tier_amd.moe_i8_layer(X.ptr, rb, S.ptr, I.ptr, W.ptr, ex.G.ptr, ex.rbg, ex.SG.ptr, ex.D.ptr, ex.rbd, ex.SD.ptr, y.ptr,
                              BF16, K, T, k, E, K, F, w_s.ptr, n, s)

    I.upload(np.full(T * k, -1, np.int32))
    graph = hip.Graph(st, lambda s: call(Y, ws, s))
    try:
        for i in range(4):
            q, sx = tokens(T, K, 20 + i)
            ids, w = routes(T, k, E, 30 + i)
            if i == 2:
                ids[0] = -1
            host = np.zeros((T, rb), np.int8)
            host[:, :K] = q
            X.upload(host), S.upload(sx), I.upload(ids), W.upload(w)
            graph.launch(st)
            st.synchronize()
            check(Y, ex, q, sx, ids, w)
            Y2 = Rows(BF16, T, K)
            call(Y2, ws2, st)
            st.synchronize()
            assert np.array_equal(Y.bits(), Y2.bits())
        assert (ws.download(np.uint8)[n:] == 0x55).all() and (ws2.download(np.uint8)[n:] == 0xff).all()
    finally:
        graph.destroy()
        st.destroy()


@pytest.mark.parametrize("T,k", [(8, 4), (30, 4), (1, 8)])
def test_two_streams(gpu, T, k):
    """Two calls at once, each with its own workspace."""
    E, K, F = 12, 512, 384
    ex, streams = Experts(E, K, F, 40), [hip.Stream(), hip.Stream()]
    n, jobs = tier_amd.moe_i8_layer_ws_bytes(T, k, K, F), []
    for i, st in enumerate(streams):
        q, sx = tokens(T, K, 41 + i)
        ids, w = routes(T, k, E, 43 + i)
        X, rb = i8_rows(q)
        jobs.append((q, sx, ids, w, X, rb, f32(sx), i32(ids), f32(w), Rows(F32, T, K), hip.DeviceBuffer(n), st))
    hip.synchronize()
    for _ in range(5):
        for q, sx, ids, w, X, rb, S, I, W, Y, ws, st in jobs:
            tier_amd.moe_i8_layer(X.ptr, rb, S.ptr, I.ptr, W.ptr, ex.G.ptr, ex.rbg, ex.SG.ptr, ex.D.ptr, ex.rbd, ex.SD.ptr,
                                  Y.ptr, F32, K, T, k, E, K, F, ws.ptr, n, st)
    hip.synchronize()
    for q, sx, ids, w, X, rb, S, I, W, Y, ws, st in jobs:
        check(Y, ex, q, sx, ids, w)
        st.destroy()


def test_layers_one_after_the_other(gpu):
    """Two layers as they are used: norm (rows for the router, codes for the experts), the routed layer, the next norm
    adding its output to the stream in place; the codes then go through a microscaled product."""
    T, k, E, K, F, N, t = 5, 2, 6, 512, 192, 96, BF16
    from mx import E2M1, E4M3, MxRows, quantize as mx_quantize, values as mx_values
    from test_gpu_norm import EPS, forward, gains
    rng = np.random.default_rng(50)
    X = Rows(t, T, K, rng.standard_normal((T, K)).astype(np.float32))
    g, exs = [gains(K, i) for i in range(3)], [Experts(E, K, F, 51 + i) for i in range(2)]
    router = rng.standard_normal((K, E))
    stream, layer_out = Rows(t, T, K, rng.standard_normal((T, K)).astype(np.float32)), X
    rb = tier_amd.i8_row_bytes(K)
    Y, Q, S = Rows(t, T, K), hip.DeviceBuffer(T * rb), hip.DeviceBuffer(T * 4)
    for i, ex in enumerate(exs):
        h, _, y = forward(t, layer_out.values(), stream.values(), g[i])
        tier_amd.rms_norm(layer_out.ptr, t, K, stream.ptr, K, f32(g[i]).ptr, EPS, stream.ptr, K, Y.ptr, K, Q.ptr, rb, S.ptr,
                          None, T, K)
        hip.synchronize()
        q, sx = quantize(y)
        assert np.array_equal(Q.download(np.int8).reshape(T, rb)[:, :K], q)
        logits = Y.values() @ router
        ids = np.argsort(-logits, 1)[:, :k].astype(np.int32)
        w = np.exp(np.take_along_axis(logits, ids, 1) / 20).astype(np.float32)
        w /= w.sum(1, keepdims=True)
        layer_out = Rows(t, T, K)
        tier_amd.moe_i8_layer(Q.ptr, rb, S.ptr, i32(ids).ptr, f32(w).ptr, ex.G.ptr, ex.rbg, ex.SG.ptr, ex.D.ptr, ex.rbd,
                              ex.SD.ptr, layer_out.ptr, t, K, T, k, E, K, F)
        hip.synchronize()
        check(layer_out, ex, q, sx, ids, w)
    _, _, y = forward(t, layer_out.values(), stream.values(), g[2])
    C, wc = MxRows(E4M3, T, K), mx_quantize(E2M1, (rng.standard_normal((N, K)) * 0.02).astype(np.float32))
    W, O = MxRows(E2M1, N, K, *wc), Rows(F32, T, N)
    tier_amd.rms_norm_mx(layer_out.ptr, t, K, stream.ptr, K, f32(g[2]).ptr, EPS, stream.ptr, K, None, 0, E4M3, C.q.ptr, C.rb,
                         C.s.ptr, C.sb, None, T, K)
    tier_amd.mx_gemm(C.q.ptr, E4M3, C.rb, C.s.ptr, C.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, None, O.ptr, F32, N, T, N, K)
    hip.synchronize()
    from test_gpu_mx import check as mx_check
    mx_check(O.values(), F32, E4M3, mx_values(E4M3, *mx_quantize(E4M3, y)), mx_values(E2M1, *wc))
