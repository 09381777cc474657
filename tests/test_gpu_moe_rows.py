"""Routed tokens to the experts and back: the plan, the rows, the weighted sum and both gradients,
against plain numpy in 64 bits.  There is no reference function (the reference refuses MoE models,
arch.py:158-159).

Whole numbers and copied rows are exact.  A sum of n fp32 products is within n + 1 unit roundoffs of
its terms' magnitudes, then one rounding to the rows' type.
"""
import numpy as np
import pytest

import tier_amd
from rows import SIZE, TINY, TYPES, UNIT, Rows, f32, i32
from tier_amd import hip

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _ids(T, k, E, how, seed=0):
    rng = np.random.default_rng(1000 * T + 10 * k + E + seed)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    if how == "drop":
        ids[rng.random((T, k)) < 0.3] = -1
        ids.ravel()[rng.integers(0, T * k)] = E
        ids.ravel()[rng.integers(0, T * k)] = np.iinfo(np.int32).max
        ids.ravel()[rng.integers(0, T * k)] = np.iinfo(np.int32).min
    elif how == "none":
        ids[:] = -1
    elif how == "one":
        ids[:] = E - 1
    return ids


def _plan(ids, E):
    """offsets, places, sorted pairs by definition."""
    flat = ids.ravel().astype(np.int64)
    live = (flat >= 0) & (flat < E)
    order = [i for i in np.argsort(np.where(live, flat, E), kind="stable") if live[i]]
    off = np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=E))]).astype(np.int32)
    srt = np.full(flat.size, -1, np.int32)
    srt[:len(order)] = order
    places = np.full(flat.size, -1, np.int32)
    places[order] = np.arange(len(order))
    return off, places.reshape(ids.shape), srt


@pytest.mark.parametrize("how", ["all", "drop", "none", "one"])
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 64), (3, 5, 7), (8, 8, 64), (511, 8, 130), (1025, 4, 40),
                                   (2048, 8, 64), (4096, 8, 3), (4099, 8, 1024), (8192, 8, 3), (8193, 8, 16), (20011, 6, 1023)])
def test_plan(gpu, T, k, E, how):
    ids = _ids(T, k, E, how)
    off, places, srt = _plan(ids, E)
    P = T * k
    skip = 4 if T % 2 else 0  # tables that start 4 bytes past a 16-byte unit
    D = hip.DeviceBuffer(4 * P + 16).upload(ids, skip)
    O, TP, SP = i32(np.full(E + 2, 77)), i32(np.full(P + 1, 77)), i32(np.full(P + 1, 77))
    n = tier_amd.moe_plan_ws_bytes(T, k, E)
    assert (n > 0) == (P > 32768)
    ws = hip.DeviceBuffer(n) if n else None
    tier_amd.moe_plan(D.ptr + skip, T, k, E, O.ptr, TP.ptr, SP.ptr, ws.ptr if ws else None, n)
    hip.synchronize()
    assert np.array_equal(O.download(np.int32), np.append(off, 77))
    assert np.array_equal(TP.download(np.int32), np.append(places.ravel(), 77))
    assert np.array_equal(SP.download(np.int32), np.append(srt, 77))


def test_plan_of_no_tokens(gpu):
    O = i32([9, 9, 9, 9])
    for T, k in ((0, 8), (5, 0)):
        tier_amd.moe_plan(None, T, k, 3, O.ptr, None, None)
        hip.synchronize()
        assert O.download(np.int32).tolist() == [0, 0, 0, 0]


# T, topk, columns, row padding, first element
SHAPES = [(1, 1, 1, 0, 0), (1, 8, 2048, 0, 0), (3, 2, 7, 0, 1), (5, 9, 129, 3, 0), (17, 8, 1408, 0, 0),
          (6, 17, 515, 5, 3), (33, 3, 5125, 0, 0), (70, 4, 256, 8, 8)]


def _case(T, k, how="drop", E=5):
    ids = _ids(T, k, E, how, seed=3)
    off, places, srt = _plan(ids, E)
    return off, places, srt, i32(places), i32(srt)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,k,K,pad,skip", SHAPES)
def test_sort_rows(gpu, t, T, k, K, pad, skip):
    rng = np.random.default_rng(K)
    _, places, srt, TP, SP = _case(T, k)
    x = rng.standard_normal((T, K)).astype(np.float32)
    x.ravel()[:3] = [np.inf, -0.0, 1e-42][:min(3, x.size)]
    X, Y = Rows(t, T, K, x, pad, skip), Rows(t, T * k, K, None, pad + 1, skip)
    tier_amd.moe_sort(X.ptr, t, X.ld, TP.ptr, SP.ptr, Y.ptr, Y.ld, T, k, K)
    hip.synchronize()
    want = np.where(srt[:, None] >= 0, X.bits()[np.maximum(srt, 0) // k], 0)
    assert np.array_equal(Y.bits(), want) and Y.outside_kept()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("T,k,N,pad,skip", SHAPES)
def test_sums_back(gpu, t, weighted, T, k, N, pad, skip):
    """unsort and the gradient of sort; dropped pairs' weights and rows hold NaN."""
    rng = np.random.default_rng(N + k)
    _, places, srt, TP, SP = _case(T, k)
    y = rng.standard_normal((T * k, N)).astype(np.float32)
    y[srt < 0] = np.nan
    w = rng.random((T, k)).astype(np.float32)
    w[places < 0] = np.nan
    Y, O, W = Rows(t, T * k, N, y, pad, skip), Rows(t, T, N, None, pad + 2, skip), f32(w)
    if weighted:
        tier_amd.moe_unsort(Y.ptr, t, Y.ld, TP.ptr, W.ptr, O.ptr, O.ld, T, k, N)
    else:
        tier_amd.moe_sort_grad(Y.ptr, t, Y.ld, TP.ptr, O.ptr, O.ld, T, k, N)
    hip.synchronize()
    live = places >= 0
    terms = np.where(live[..., None], Y.values()[np.maximum(places, 0)], 0.0)
    if weighted:
        terms = terms * np.where(live, w, 0).astype(np.float64)[..., None]
    want, mag = terms.sum(1), np.abs(terms).sum(1)
    err = (k + 1) * U * mag
    assert np.all(np.abs(O.values() - want) <= err + UNIT[t] * (np.abs(want) + err) + TINY[t])
    assert O.outside_kept()


def _unsort_grad(t, T, k, N, pad=0, skip=0, seed=0, how="drop"):
    rng = np.random.default_rng(N + k + seed)
    _, places, srt, TP, SP = _case(T, k, how)
    y = rng.standard_normal((T * k, N)).astype(np.float32)
    w = rng.random((T, k)).astype(np.float32)
    y[srt < 0] = np.nan
    w[places < 0] = np.nan
    d = rng.standard_normal((T, N)).astype(np.float32)
    D, Y, W = Rows(t, T, N, d, pad, skip), Rows(t, T * k, N, y, pad + 1, skip), f32(w)
    DY, DW = Rows(t, T * k, N, None, pad + 2, skip), f32(np.full(T * k + 1, 5.0))
    tier_amd.moe_unsort_grad(D.ptr, t, D.ld, Y.ptr, Y.ld, TP.ptr, SP.ptr, W.ptr, DY.ptr, DY.ld, DW.ptr, T, k, N)
    hip.synchronize()
    dw = DW.download(np.float32)
    assert dw[-1] == 5.0 and DY.outside_kept()
    return places, srt, D.values(), Y.values(), w, DY.values(), dw[:-1].reshape(T, k).astype(np.float64)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,k,N,pad,skip", SHAPES + [(600, 8, 96, 0, 0), (2100, 2, 513, 0, 0)])
def test_unsort_grad(gpu, t, T, k, N, pad, skip):
    places, srt, d, y, w, dy, dw = _unsort_grad(t, T, k, N, pad, skip)
    live = srt >= 0
    i = np.maximum(srt, 0)
    want = np.where(live[:, None], np.where(live, w.ravel()[i], 0).astype(np.float64)[:, None] * d[i // k], 0.0)
    assert np.all(np.abs(dy - want) <= (U + UNIT[t] * (1 + U)) * np.abs(want) + TINY[t])
    here = places >= 0
    terms = np.where(here[..., None], d[:, None] * y[np.maximum(places, 0)], 0.0)
    # a thread's chain of its columns, the wave's and the workgroup's sums
    n = -(-N // 256) + 8 + 8
    assert np.all(np.abs(dw - terms.sum(-1)) <= n * U * np.abs(terms).sum(-1))
    assert np.all(dw[~here] == 0)


def test_gradients_are_those_of_the_sums(gpu):
    """Differences of L = <dout, unsort(Ys, w)> along directions of Ys and of w, and of <g, sort(x)>:
    both are linear in each, so a step of 1/4 has no truncation, only the sums' roundings."""
    t, T, k, N, h = tier_amd.F32, 37, 4, 130, 0.25
    places, srt, d, y, w, dy, dw = _unsort_grad(t, T, k, N)
    rng = np.random.default_rng(8)
    vy, vw = rng.standard_normal(y.shape), rng.standard_normal(w.shape)
    y0, w0 = np.nan_to_num(y), np.nan_to_num(w).astype(np.float64)
    TP, SP = i32(places), i32(srt)

    def out(yy, ww):
        Y, O, W = Rows(t, T * k, N, yy), Rows(t, T, N), f32(ww)
        tier_amd.moe_unsort(Y.ptr, t, N, TP.ptr, W.ptr, O.ptr, N, T, k, N)
        hip.synchronize()
        return O.values()

    big = np.abs(d).sum() * (1 + np.abs(y0).max() + h * np.abs(vy).max()) * (1 + h * np.abs(vw).max()) * k
    tol = 2 * (k + 4) * U * big / (2 * h)  # both ends' sums and their rounded inputs
    got = (d * (out(y0 + h * vy, w0) - out(y0 - h * vy, w0))).sum() / (2 * h)
    assert abs(got - (dy * vy).sum()) <= tol
    got = (d * (out(y0, w0 + h * vw) - out(y0, w0 - h * vw))).sum() / (2 * h)
    assert abs(got - (dw * vw).sum()) <= tol

    g, x, vx = (rng.standard_normal(s) for s in ((T * k, N), (T, N), (T, N)))

    def rows(xx):
        X, Y = Rows(t, T, N, xx), Rows(t, T * k, N)
        tier_amd.moe_sort(X.ptr, t, N, TP.ptr, SP.ptr, Y.ptr, N, T, k, N)
        hip.synchronize()
        return Y.values()

    G, DX = Rows(t, T * k, N, g), Rows(t, T, N)
    tier_amd.moe_sort_grad(G.ptr, t, N, TP.ptr, DX.ptr, N, T, k, N)
    hip.synchronize()
    got = (G.values() * (rows(x + h * vx) - rows(x - h * vx))).sum() / (2 * h)
    tol = 2 * (k + 4) * U * np.abs(g).sum() * (np.abs(x).max() + np.abs(vx).max()) / (2 * h)
    assert abs(got - (DX.values() * vx).sum()) <= tol


def test_all_dropped(gpu):
    t, T, k, N = tier_amd.F32, 4, 3, 40
    places, srt, d, y, w, dy, dw = _unsort_grad(t, T, k, N, how="none")
    assert np.all(dy == 0) and np.all(dw == 0)
    Y, O, W = Rows(t, T * k, N, np.full((T * k, N), np.nan)), Rows(t, T, N), f32(np.full((T, k), np.nan))
    tier_amd.moe_unsort(Y.ptr, t, N, i32(places).ptr, W.ptr, O.ptr, N, T, k, N)
    hip.synchronize()
    assert np.all(O.values() == 0)


def test_places_out_of_range_are_dropped(gpu):
    """Tables that do not come from the plan: places past the rows are not followed."""
    t, T, k, N = tier_amd.F16, 2, 2, 24
    places = np.array([[0, 99], [-5, 3]], np.int32)
    TP, SP, W = i32(places), i32([0, -1, -1, 3]), f32([[1, 2], [3, 4]])
    x = np.arange(T * N).reshape(T, N)
    X, Y = Rows(t, T, N, x), Rows(t, T * k, N)
    tier_amd.moe_sort(X.ptr, t, N, TP.ptr, SP.ptr, Y.ptr, N, T, k, N)
    O = Rows(t, T, N)
    tier_amd.moe_unsort(Y.ptr, t, N, TP.ptr, W.ptr, O.ptr, N, T, k, N)
    hip.synchronize()
    assert np.array_equal(Y.values(), np.stack([x[0], 0 * x[0], 0 * x[0], x[1]]).astype(float))
    assert np.array_equal(O.values(), np.stack([x[0], 4 * x[1]]).astype(float))


def test_on_a_stream_and_in_a_graph(gpu):
    """The layer's way there and back on a stream of its own, captured once: replays follow the ids."""
    t, T, k, E, K = tier_amd.F32, 19, 3, 6, 200
    rng = np.random.default_rng(4)
    x, w = rng.standard_normal((T, K)).astype(np.float32), rng.random((T, k)).astype(np.float32)
    X, Y, O, W = Rows(t, T, K, x), Rows(t, T * k, K), Rows(t, T, K), f32(w)
    D, OF, TP, SP = i32(_ids(T, k, E, "all")), i32(np.zeros(E + 1)), i32(np.zeros(T * k)), i32(np.zeros(T * k))

    def step(s):
        tier_amd.moe_plan(D.ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr, stream=s)
        tier_amd.moe_sort(X.ptr, t, K, TP.ptr, SP.ptr, Y.ptr, K, T, k, K, stream=s)
        tier_amd.moe_unsort(Y.ptr, t, K, TP.ptr, W.ptr, O.ptr, K, T, k, K, stream=s)

    s = hip.Stream()
    g = hip.Graph(s, step)
    for n in range(4):
        ids = _ids(T, k, E, "drop", seed=n)
        D.upload(ids)
        hip.synchronize()
        g.launch(s)
        s.synchronize()
        off, places, srt = _plan(ids, E)
        assert np.array_equal(OF.download(np.int32), off) and np.array_equal(SP.download(np.int32), srt)
        replayed = O.bits().copy()
        want = x * np.where(places >= 0, w, 0).astype(np.float64).sum(1)[:, None]
        assert np.all(np.abs(O.values() - want) <= (k + 1) * U * np.abs(want))
        step(s)
        s.synchronize()
        assert np.array_equal(O.bits(), replayed)
    g.destroy()
    s.destroy()


def test_rows_past_the_caches(gpu):
    """Gathered rows of more bytes than the caches keep (80 MiB) take the streaming form of the sums."""
    t, T, k, N = tier_amd.F32, 2500, 8, 1050
    rng = np.random.default_rng(1)
    _, places, srt, TP, SP = _case(T, k, E=16)
    y = rng.standard_normal((T * k, N)).astype(np.float32)
    w = rng.random((T, k)).astype(np.float32)
    Y, O, G, W = Rows(t, T * k, N, y, pad=2), Rows(t, T, N), Rows(t, T, N), f32(w)
    tier_amd.moe_unsort(Y.ptr, t, Y.ld, TP.ptr, W.ptr, O.ptr, N, T, k, N)
    tier_amd.moe_sort_grad(Y.ptr, t, Y.ld, TP.ptr, G.ptr, N, T, k, N)
    hip.synchronize()
    live = places >= 0
    rows = np.where(live[..., None], y[np.maximum(places, 0)], np.float32(0)).astype(np.float64)
    for got, terms in ((O, rows * np.where(live, w, 0).astype(np.float64)[..., None]), (G, rows)):
        want, mag = terms.sum(1), np.abs(terms).sum(1)
        assert np.all(np.abs(got.values() - want) <= (k + 2) * U * mag)


def test_row_offsets_past_32_bits(gpu):
    """Rows 32 MiB apart: the last ones start past 4 GiB."""
    t, T, k, N, ld = tier_amd.F16, 2, 70, 24, 1 << 24
    P, rng = T * k, np.random.default_rng(2)
    _, places, srt, TP, SP = _case(T, k, how="drop", E=5)
    x, w, d = (rng.standard_normal(s).astype(np.float32) for s in ((T, N), (T, k), (T, N)))
    X, D, O, W, DW = Rows(t, T, N, x), Rows(t, T, N, d), Rows(t, T, N), f32(w), f32(np.zeros(P))
    far, far2 = hip.DeviceBuffer((P - 1) * ld * 2 + 64), hip.DeviceBuffer((P - 1) * ld * 2 + 64)
    rows = lambda b: np.stack([b.download(np.float16, N, p * ld * 2) for p in range(P)]).astype(np.float64)  # noqa: E731
    tier_amd.moe_sort(X.ptr, t, N, TP.ptr, SP.ptr, far.ptr, ld, T, k, N)
    tier_amd.moe_unsort(far.ptr, t, ld, TP.ptr, W.ptr, O.ptr, N, T, k, N)
    tier_amd.moe_unsort_grad(D.ptr, t, N, far.ptr, ld, TP.ptr, SP.ptr, W.ptr, far2.ptr, ld, DW.ptr, T, k, N)
    hip.synchronize()
    xs, i = X.values(), np.maximum(srt, 0)
    assert np.array_equal(rows(far), np.where(srt[:, None] >= 0, xs[i // k], 0))
    live = places >= 0
    terms = np.where(live, w, 0).astype(np.float64)[..., None] * xs[:, None]
    err = (k + 1) * U * np.abs(terms).sum(1)
    assert np.all(np.abs(O.values() - terms.sum(1)) <= err + UNIT[t] * (np.abs(terms.sum(1)) + err) + TINY[t])
    want = np.where(srt[:, None] >= 0, w.ravel()[i].astype(np.float64)[:, None] * D.values()[i // k], 0)
    assert np.all(np.abs(rows(far2) - want) <= (U + UNIT[t] * (1 + U)) * np.abs(want) + TINY[t])
    dots = D.values() * xs
    dw = DW.download(np.float32).reshape(T, k)
    assert np.all(np.abs(dw - np.where(live, dots.sum(1)[:, None], 0)) <= 17 * U * np.abs(dots).sum(1)[:, None])
