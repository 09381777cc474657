"""The plan's tables in the entry points that were there before it: tiermm_qgemm_grouped (from a host
copy of the offsets) on the rows of tiermm_moe_sort, and tiermm_moe_combine with the weights in
sorted order; also where pairs are dropped.

The experts' products are held to the grouped GEMM's own bar (relative Frobenius error 2^-20); a
combined value is a sum of topk fp32 products of the rows that the device holds: topk + 1 unit
roundoffs of its terms' magnitudes.
"""
import numpy as np
import pytest

import oracle
import tier_amd
from rows import Rows, f32, i32
from tier_amd import hip

pytestmark = pytest.mark.gpu
U, BAR = 2.0 ** -24, 2.0 ** -20


# N % 4 != 0 and topk > 16 take the combine's general kernel
@pytest.mark.parametrize("N,T,topk,drop", [(256, 50, 2, 0.0), (256, 50, 2, 0.3), (192, 33, 16, 0.5), (130, 21, 3, 0.4),
                                           (64, 9, 20, 0.5), (128, 5, 4, 1.0)])
def test_plan_feeds_grouped_gemm_and_combine(gpu, N, T, topk, drop):
    t, E, K, P = tier_amd.Q4_K, 6, 512, T * topk
    rng = np.random.default_rng(N + T)
    ids = rng.integers(0, E, (T, topk)).astype(np.int32)
    ids[rng.random((T, topk)) < drop] = -1
    x = rng.standard_normal((T, K)).astype(np.float32)
    w = rng.random((T, topk)).astype(np.float32)
    blocks = [oracle.random_blocks(rng, t, N * (K // oracle.block(t)[0])).reshape(N, -1) for _ in range(E)]
    dW, rb = [hip.to_device(b) for b in blocks], tier_amd.q_row_bytes(t, K)

    OF, TP, SP = i32(np.zeros(E + 1)), i32(np.zeros(P)), i32(np.zeros(P))
    tier_amd.moe_plan(i32(ids).ptr, T, topk, E, OF.ptr, TP.ptr, SP.ptr)
    X, XS = Rows(tier_amd.F32, T, K, x), Rows(tier_amd.F32, P, K)
    tier_amd.moe_sort(X.ptr, tier_amd.F32, K, TP.ptr, SP.ptr, XS.ptr, K, T, topk, K)
    hip.synchronize()
    off, places, order = OF.download(np.int32), TP.download(np.int32), SP.download(np.int32)
    # places without a pair hold NaN, rows of Y and weights: nothing of them may enter a sum
    Y = Rows(tier_amd.F32, P, N, np.full((P, N), np.nan))
    tier_amd.qgemm_grouped([b.ptr for b in dW], [t] * E, [rb] * E, XS.ptr, off.tolist(), Y.ptr, N, K)
    sorted_w = np.where(order >= 0, w.ravel()[np.maximum(order, 0)], np.float32(np.nan))
    OUT = Rows(tier_amd.F32, T, N, np.full((T, N), 7.0))
    tier_amd.moe_combine(Y.ptr, TP.ptr, f32(sorted_w).ptr, OUT.ptr, T, topk, N)
    hip.synchronize()

    y = Y.values()
    assert np.isnan(y[off[E]:]).all()
    want = np.empty((off[E], N))
    for e in range(E):
        r = order[off[e]:off[e + 1]]
        w16 = oracle.h2f(oracle.dequant(blocks[e], t, K, oracle.OUT_F16)).reshape(N, K).astype(np.float64)
        want[off[e]:off[e + 1]] = x[r // topk].astype(np.float64) @ w16.T
    if off[E]:
        assert oracle.rel_fro(y[:off[E]], want) <= BAR
    live = (places >= 0).reshape(T, topk)
    at = np.maximum(places, 0).reshape(T, topk)
    terms = np.where(live[..., None], y[at] * w.astype(np.float64)[..., None], 0.0)
    assert np.all(np.abs(OUT.values() - terms.sum(1)) <= (topk + 1) * U * np.abs(terms).sum(1))
