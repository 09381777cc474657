"""A routed layer of few pairs: a result's bits are the same in every call."""
import numpy as np
import pytest

from test_gpu_moe_layer import Experts, routes, run, tokens

pytestmark = pytest.mark.gpu


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
