"""int8 products where tables, scales and codes are unusual: a slice of the experts, rows that point
nowhere, scales at the ends of fp32, codes of -128; and every kernel variant with a bias, in every
type.  Bounds as in test_gpu_i8.py."""
import numpy as np
import pytest

import tier_amd
from rows import TYPES, Rows, f32, i32
from test_gpu_i8 import _routed, check, i8_rows, weight
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
