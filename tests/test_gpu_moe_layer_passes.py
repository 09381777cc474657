"""A routed layer of few pairs whose fullest expert has more of them than its down kernel takes at a time (8): the
passes' shared memory and the counters of replayed calls; and that a result's bits are the same in every call.
"""
import numpy as np
import pytest

import tier_amd
from rows import Rows
from test_gpu_i8 import i8_rows
from test_gpu_moe_layer import Experts, check, routes, run, tokens
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, F16, BF16 = tier_amd.F32, tier_amd.F16, tier_amd.BF16


def crowded(T, k, E, n, seed):
    """Routes of T tokens in which expert E - 1 has n pairs, no token naming it twice."""
    rng = np.random.default_rng(seed)
    ids = np.argsort(rng.random((T, E - 1)), 1)[:, :k].astype(np.int32) if E > k else rng.integers(0, E - 1, (T, k)).astype(np.int32)
    for t in rng.choice(T, min(n, T), replace=False):
        ids[t, rng.integers(0, k)] = E - 1
    w = rng.random((T, k)).astype(np.float32)
    return ids, w / w.sum(1, keepdims=True)


@pytest.mark.parametrize("F", [96, 1408])
@pytest.mark.parametrize("T,k,E,n", [(32, 1, 4, 32), (32, 1, 40, 32), (16, 2, 5, 9), (16, 2, 48, 16), (17, 1, 3, 17),
                                     (32, 1, 64, 25), (10, 3, 4, 10), (8, 4, 33, 8)])
def test_more_pairs_than_a_pass_takes(gpu, T, k, E, n, F):
    K = 136
    ex = Experts(E, K, F, T + E)
    q, sx = tokens(T, K, T)
    ids, w = crowded(T, k, E, n, n)
    assert T * k <= 32 and (ids == E - 1).sum() == n
    for t in (F32, BF16):
        check(run(ex, q, sx, ids, w, t), ex, q, sx, ids, w)


@pytest.mark.parametrize("T,k", [(32, 1), (16, 2)])
def test_all_pairs_on_one_expert(gpu, T, k):
    E, K, F = 3, 200, 1408
    ex = Experts(E, K, F, 5)
    q, sx = tokens(T, K, 6)
    ids, w = np.full((T, k), 1, np.int32), np.random.default_rng(7).random((T, k)).astype(np.float32)
    check(run(ex, q, sx, ids, w, F16), ex, q, sx, ids, w)
    ids[T // 2, 0] = 9  # dropped
    check(run(ex, q, sx, ids, w), ex, q, sx, ids, w)


def test_captured_through_passes(gpu):
    """One graph: all pairs on one expert, then spread ones, then all on another, against eager calls in turn."""
    T, k, E, K, F, st = 16, 2, 12, 256, 1408, hip.Stream()
    ex = Experts(E, K, F, 13)
    X, rb = i8_rows(np.zeros((T, K), np.int64))
    S, I, W, Y = hip.DeviceBuffer(T * 4), hip.DeviceBuffer(T * k * 4), hip.DeviceBuffer(T * k * 4), Rows(F32, T, K)
    n = tier_amd.moe_i8_layer_ws_bytes(T, k, K, F)
    ws, ws2 = hip.DeviceBuffer(n), hip.DeviceBuffer(n)
    ws.fill_bytes(0x55), ws2.fill_bytes(0xff)

    def call(y, w_s, s):
        tier_amd.moe_i8_layer(X.ptr, rb, S.ptr, I.ptr, W.ptr, ex.G.ptr, ex.rbg, ex.SG.ptr, ex.D.ptr, ex.rbd, ex.SD.ptr, y.ptr,
                              F32, K, T, k, E, K, F, w_s.ptr, n, s)

    I.upload(np.full(T * k, -1, np.int32))
    graph = hip.Graph(st, lambda s: call(Y, ws, s))
    try:
        for i, ids in enumerate((np.full((T, k), 4), routes(T, k, E, 1)[0], crowded(T, k, E, 11, 2)[0], np.full((T, k), 11))):
            q, sx = tokens(T, K, 20 + i)
            w = np.random.default_rng(i).random((T, k)).astype(np.float32)
            host = np.zeros((T, rb), np.int8)
            host[:, :K] = q
            X.upload(host), S.upload(sx), I.upload(ids.astype(np.int32)), W.upload(w)
            graph.launch(st)
            st.synchronize()
            check(Y, ex, q, sx, ids, w)
            Y2 = Rows(F32, T, K)
            call(Y2, ws2, st)
            st.synchronize()
            assert np.array_equal(Y.bits(), Y2.bits())
    finally:
        graph.destroy()
        st.destroy()


def test_sign_of_underflow_does_not_depend_on_the_call(gpu):
    """Products with weights so small that fp32 has only a zero for them: the zero's sign is the token's own, whether
    it comes alone or with 39 others."""
    E, K, F, T = 3, 140, 64, 40
    ex = Experts(E, K, F, 15)
    q, sx = tokens(T, K, 16)
    ids, w = routes(T, 1, E, 17)
    w[:] = np.float32(2.0 ** -149)
    whole = run(ex, q, sx * np.float32(1e-4), ids, w).bits()
    assert (whole == 0x80000000).any() and (whole == 0).any()
    alone = [run(ex, q[i:i + 1], sx[i:i + 1] * np.float32(1e-4), ids[i:i + 1], w[i:i + 1]).bits() for i in range(T)]
    assert np.array_equal(np.concatenate(alone), whole)
