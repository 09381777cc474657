"""int8 products where tables, scales and codes are unusual: a slice of the experts, rows that point
nowhere, scales at the ends of fp32, codes of -128; and every kernel variant with a bias, in every
type.  Bounds as in test_gpu_i8.py."""
import numpy as np
import pytest

import tier_amd
from rows import TINY, TYPES, UNIT, Rows, f32, i32
from test_gpu_i8 import _routed, check, i8_rows, quantize, weight
from tier_amd import hip

pytestmark = pytest.mark.gpu

# T, topk, experts, N, K: tiles of 16, 64 and 128 to 256 rows
GROUPED = [(9, 4, 12, 96, 256), (200, 1, 9, 1010, 130), (500, 1, 9, 3500, 130), (3000, 3, 33, 300, 512),
           (1100, 2, 3, 1000, 260)]


@pytest.mark.parametrize("T,k,E,N,K", GROUPED)
def test_grouped_slice_of_experts(gpu, T, k, E, N, K):
    """Experts e0 .. e1 - 1 of a plan: the offsets start above 0, and rows on both sides become zeros."""
    t, P = tier_amd.F32, T * k
    ids = _routed(T, k, E, T, drop=0.1)
    q = np.random.default_rng(N).integers(-127, 128, (T, K))
    X, rb = i8_rows(q)
    sx = np.random.default_rng(T).random(T).astype(np.float32)
    w, sw, W, rbw = weight(E * N, K, 13)
    OF, TP, SP, SW = i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P)), f32(sw)
    tier_amd.moe_plan(i32(ids).ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr)
    for e0, e1 in ((1, E), (E // 2, E - 1), (E - 1, E)):
        Y = Rows(t, P, N, np.full((P, N), np.nan))
        tier_amd.i8_gemm_grouped(X.ptr, rb, f32(sx).ptr, SP.ptr, T, k, OF.ptr + 4 * e0, e1 - e0, W.ptr + e0 * N * rbw,
                                 rbw, SW.ptr + 4 * e0 * N, Y.ptr, t, N, P, N, K)
        hip.synchronize()
        off, srt, y = OF.download(np.int32), SP.download(np.int32), Y.values()
        assert not y[:off[e0]].any() and not y[off[e1]:].any()
        for e in range(e0, e1):
            r = srt[off[e]:off[e + 1]] // k
            check(y[off[e]:off[e + 1]], t, q[r], sx[r], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])


def test_grouped_without_rows_of_its_experts(gpu):
    """All rows in front of the first offset, or all behind the last."""
    t, E, N, K, P = tier_amd.BF16, 3, 70, 130, 40
    X, rb = i8_rows(np.ones((P, K), np.int64))
    w, sw, W, rbw = weight(E * N, K, 1)
    for at in (0, P):
        Y = Rows(t, P, N, np.full((P, N), np.nan))
        tier_amd.i8_gemm_grouped(X.ptr, rb, f32(np.ones(P)).ptr, None, P, 1, i32([at] * (E + 1)).ptr, E, W.ptr, rbw,
                                 f32(sw).ptr, Y.ptr, t, N, P, N, K)
        hip.synchronize()
        assert not Y.values().any()


# rows of x: the GEMV, the small tiles, 64 x 64, 128 x 128 and 256-row tiles
ROWS = [(1, 300, 640), (2, 300, 640), (6, 1003, 260), (50, 2501, 260), (50, 5101, 2600), (130, 20001, 130),
        (2051, 2001, 130)]


@pytest.mark.parametrize("t", [tier_amd.F32, tier_amd.BF16])
@pytest.mark.parametrize("M,N,K", ROWS)
def test_scales_at_the_ends_of_fp32(gpu, t, M, N, K):
    """sx * sw below the normal numbers or past the largest one, while the element is not: within the
    same bound, and a sum of 0 gives the bias.  Elements that are too large themselves are infinite."""
    rng = np.random.default_rng(M + N)
    q = rng.integers(-127, 128, (M, K))
    if M > 2:
        q[M // 2] = 0
    sx = np.float32([2.0 ** -120, 2.0 ** 100, 1, 2.0 ** -149, 3 * 2.0 ** -130, 2.0 ** 120, 2.0 ** -64])[rng.permutation(M) % 7]
    w, _, W, rbw = weight(N, K, M + N)
    sw = np.float32([2.0 ** -11, 2.0 ** 20, 2.0 ** -60, 2.0 ** 110, 2.0 ** -126, 3, 2.0 ** 63])[rng.permutation(N) % 7]
    sw *= rng.choice(np.float32([-1, 1]), N)
    bias = np.where(rng.random(N) < 0.5, 0, rng.standard_normal(N)).astype(np.float32)
    X, rbx = i8_rows(q)
    Y = Rows(t, M, N)
    tier_amd.i8_gemm(X.ptr, rbx, f32(sx).ptr, W.ptr, rbw, f32(sw).ptr, f32(bias).ptr, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    y = Y.values()
    s = (q.astype(np.float64) @ w.T.astype(np.float64)) * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    top = 2.0 ** 128 * (1 - 2.0 ** -7)  # (bf16 and roundings at the very end are left out)
    large, fits = np.abs(s) >= 2.0 ** 128 * (1 + 2.0 ** -20), np.abs(s) < top
    assert np.array_equal(y[large], np.where(s > 0, np.inf, -np.inf)[large])
    err = 4 * 2.0 ** -24 * (np.abs(s) + np.abs(bias))
    unit, tiny = UNIT[t], TINY[tier_amd.F32] + TINY[t]
    ok = np.abs(y - (s + bias)) <= err + unit * (np.abs(s + bias) + err) + tiny
    assert ok[fits].all(), np.argwhere(~ok & fits)[:5]
    if M > 2:
        assert not s[M // 2].any() and large.any() and (np.abs(s[s != 0]) < 2.0 ** -126).any()


@pytest.mark.parametrize("M", [1, 2, 5, 40, 150])
@pytest.mark.parametrize("down", [100, 120, 130])
def test_linear_of_tiny_rows(gpu, M, down):
    """Rows of x of 2^-down times normal numbers: products of their codes to the same bound."""
    t, N, K = tier_amd.F32, 200, 700
    x = np.random.default_rng(M).standard_normal((M, K)).astype(np.float32) * np.float32(2.0 ** -down)
    w, sw, W, rbw = weight(N, K, 4)
    sw *= np.float32(2.0 ** 10)
    X, Y = Rows(t, M, K, x), Rows(t, M, N)
    tier_amd.i8_linear(X.ptr, t, K, W.ptr, rbw, f32(sw).ptr, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    q, sx = quantize(x)
    check(Y.values(), t, q, sx, w, sw)


def test_grouped_scales_at_the_ends_of_fp32(gpu):
    """The same of the experts' products, where one token's scale is tiny."""
    t, T, k, E, N, K = tier_amd.F32, 600, 2, 3, 520, 260
    q = np.random.default_rng(1).integers(-127, 128, (T, K))
    X, rb = i8_rows(q)
    sx = np.float32([1, 2.0 ** -125, 2.0 ** 70])[np.arange(T) % 3]
    w, sw, W, rbw = weight(E * N, K, 3)
    P = T * k
    OF, TP, SP, Y = i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P)), Rows(t, P, N)
    tier_amd.moe_plan(i32(_routed(T, k, E, 5)).ptr, T, k, E, OF.ptr, TP.ptr, SP.ptr)
    tier_amd.i8_gemm_grouped(X.ptr, rb, f32(sx).ptr, SP.ptr, T, k, OF.ptr, E, W.ptr, rbw, f32(sw).ptr, Y.ptr, t, N, P, N, K)
    hip.synchronize()
    off, srt, y = OF.download(np.int32), SP.download(np.int32), Y.values()
    for e in range(E):
        r = srt[off[e]:off[e + 1]] // k
        check(y[off[e]:off[e + 1]], t, q[r], sx[r], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("P,E,N,K", [(9, 3, 70, 130), (40, 3, 1010, 130), (500, 9, 3500, 130), (3000, 33, 300, 512),
                                     (2200, 3, 1000, 260)])
def test_rows_that_point_nowhere(gpu, t, P, E, N, K):
    """Indices below 0 and past the rows of x: zeros, also in channels whose scale is NaN or infinite,
    where every other row is not finite."""
    rng = np.random.default_rng(P)
    T, topk = P // 2 + 1, 2
    q = rng.integers(1, 128, (T, K))
    X, rb = i8_rows(q)
    w, sw, W, rbw = weight(E * N, K, 2)
    w = np.abs(w) + (w == 0)  # sums above 0
    W, rbw = i8_rows(w)
    bad = rng.random(E * N) < 0.02
    bad[::N] = True
    sw[bad] = rng.choice(np.float32([np.nan, np.inf, -np.inf]), bad.sum())
    rows = rng.integers(0, T * topk, P).astype(np.int32)
    rows[rng.random(P) < 0.2] = -1
    rows[rng.random(P) < 0.1] = T * topk
    rows[:2] = [np.iinfo(np.int32).min, np.iinfo(np.int32).max]
    off = np.sort(rng.integers(0, P + 1, E + 1)).astype(np.int32)
    off[0], off[E] = 0, P
    sx = rng.random(T).astype(np.float32)
    Y = Rows(t, P, N, np.full((P, N), 5.0))
    tier_amd.i8_gemm_grouped(X.ptr, rb, f32(sx).ptr, i32(rows).ptr, T, topk, i32(off).ptr, E, W.ptr, rbw, f32(sw).ptr,
                             Y.ptr, t, N, P, N, K)
    hip.synchronize()
    y = Y.values()
    nowhere = (rows < 0) | (rows >= T * topk)
    assert not y[nowhere].any()
    for e in range(E):
        at = np.arange(off[e], off[e + 1])
        at = at[~nowhere[at]]
        r, c, b = rows[at] // topk, slice(e * N, (e + 1) * N), bad[e * N:(e + 1) * N]
        assert not np.isfinite(y[at][:, b]).any()
        if t != tier_amd.F16:  # (fp16 does not hold these sums)
            check(y[at][:, ~b], t, q[r], sx[r], w[c][~b], sw[c][~b])


@pytest.mark.parametrize("M", [1, 3, 20, 140])
@pytest.mark.parametrize("x,K", [(127, 132104), (-127, 132104), (-128, 131071)])
def test_largest_sums_with_codes_of_128(gpu, M, x, K):
    """Weights of -128 all over against the codes of largest magnitude, at the largest K that the header
    states for them: the sums are 2^31 - 1024 and thereabouts, and exact."""
    N, t = 3, tier_amd.F32
    assert abs(x) * 128 * K < 2 ** 31 <= abs(x) * 128 * (K + 1)
    w = np.full((N, K), -128, np.int64)
    w[1] = 127
    q = np.full((M, K), x, np.int64)
    W, rbw = i8_rows(w)
    X, rbx = i8_rows(q)
    one, Y = np.ones(M, np.float32), Rows(t, M, N)
    tier_amd.i8_gemm(X.ptr, rbx, f32(one).ptr, W.ptr, rbw, f32(np.ones(N)).ptr, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    check(Y.values(), t, q, one, w, np.ones(N, np.float32))
    # and of an expert's rows
    Z = Rows(t, M, N)
    tier_amd.i8_gemm_grouped(X.ptr, rbx, f32(one).ptr, None, M, 1, i32([0, M]).ptr, 1, W.ptr, rbw, f32(np.ones(N)).ptr,
                             Z.ptr, t, N, M, N, K)
    hip.synchronize()
    assert np.array_equal(Y.bits(), Z.bits())
