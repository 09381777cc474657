"""x3-ref weights are fp16(fp32 value), rounded twice as the dequant rounds them: weights whose fp32
value lies on a tie of fp16 that the exact value does not (rounded once, such a weight is one fp16 step
off).  Unit vectors, so every product is one weight and the bits have to be equal."""
import numpy as np
import pytest

import oracle
import tier_amd
from rows import Rows
from tier_amd import hip

pytestmark = pytest.mark.gpu


def _exact(blocks, t, K):
    """q4_K / q5_K rows in 64 bits: d sc q - dmin mn, without a rounding."""
    b = blocks.reshape(-1, oracle.block(t)[1])
    h = b[:, :4].copy().view(np.float16).astype(np.float64)
    s = b[:, 4:16].astype(np.int64)
    lo, hi, top = s[:, 0:4], s[:, 4:8], s[:, 8:12]
    sc = np.concatenate([lo & 63, (top & 15) | ((lo >> 6) << 4)], 1)
    mn = np.concatenate([hi & 63, (top >> 4) | ((hi >> 6) << 4)], 1)
    n = b[:, -128:].astype(np.int64).reshape(-1, 4, 32)
    q = np.stack([n & 15, n >> 4], 2).reshape(-1, 8, 32)
    if t == tier_amd.Q5_K:
        q += ((b[:, 16:48].astype(np.int64)[:, None, :] >> np.arange(8)[:, None]) & 1) << 4
    w = h[:, :1, None] * sc[..., None] * q - h[:, 1:, None] * mn[..., None]
    return w.reshape(-1, K)


@pytest.mark.parametrize("M", [1, 2, 16, 32, 48, 200])
@pytest.mark.parametrize("t", [tier_amd.Q4_K, tier_amd.Q5_K])
def test_weights_on_fp16_ties(gpu, t, M):
    N, K = 3000, 1024
    rng = np.random.default_rng(t)
    blocks = oracle.random_blocks(rng, t, N * K // 256).reshape(N, -1)
    want = oracle.h2f(oracle.dequant(blocks, t, K, oracle.OUT_F16)).reshape(N, K)
    once = _exact(blocks, t, K).astype(np.float16).astype(np.float32)
    ties = np.unique(np.argwhere(once != want)[:, 1])  # their columns
    assert len(ties)
    W, rb = hip.to_device(blocks), tier_amd.q_row_bytes(t, K)
    for i in range(0, len(ties), M):
        c = np.resize(ties[i:i + M], M)
        x = np.zeros((M, K), np.float32)
        x[np.arange(M), c] = 1.0
        X, Y = Rows(tier_amd.F32, M, K, x), Rows(tier_amd.F32, M, N)
        tier_amd.qgemm(W.ptr, t, rb, X.ptr, Y.ptr, M, N, K, N, tier_amd.MODE_X3REF)
        hip.synchronize()
        assert np.array_equal(Y.values(), want[:, c].T.astype(np.float64))
