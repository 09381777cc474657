"""Every tile of the microscaled products: sizes at which each of the three cost tables takes each of its tiles on 256
CUs, with partly filled ones at the ends, one stage and several; rows far apart and past 32 bits.  Bounds as in
test_gpu_mx.py, on all columns of the first, the last and some other rows."""
import numpy as np
import pytest

import mx
import tier_amd
from mx import E2M1, E4M3, MxRows
from rows import TINY, UNIT, Rows, f32
from test_gpu_mx import check
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, BF16 = tier_amd.F32, tier_amd.BF16


def random_rows(fmt, rows, K, seed):
    """Codes of every kind and scales of some range."""
    rng = np.random.default_rng(seed)
    c = rng.integers(0, 1 << fmt, (rows, K), dtype=np.uint8).astype(np.int64)
    if fmt == E4M3:
        c = np.where(c & 127 == 127, 5, c)
    return c, rng.integers(120, 132, (rows, -(-K // 32)))


def some_rows(M, seed):
    r = np.random.default_rng(seed).integers(0, M, 20)
    return np.unique(np.concatenate([r, [0, M - 1, M // 2]]))


SIZES = [(17, 33), (2000, 33), (65, 3200), (2050, 33), (2050, 101), (2050, 250), (2050, 503), (2050, 1000), (1300, 3200),
         (2000, 3200), (2050, 4003), (1025, 7000), (1025, 10001), (1025, 14000)]


def every_output(M, N, K):
    wc, ws = random_rows(E2M1, N, K, N + K)
    W, w = MxRows(E2M1, N, K, wc, ws), mx.values(E2M1, wc, ws)
    bias = np.random.default_rng(1).standard_normal(N).astype(np.float32) * 100
    B, pick = f32(bias), some_rows(M, N)
    for xfmt in (E2M1, E4M3):
        c, s = random_rows(xfmt, M, K, M + K + xfmt)
        X, x = MxRows(xfmt, M, K, c, s), mx.values(xfmt, c[pick], s[pick])
        for t in (F32, BF16):
            Y = Rows(t, M, N, pad=1, skip=1)
            tier_amd.mx_gemm(X.q.ptr, xfmt, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, B.ptr, Y.ptr, t, Y.ld, M, N, K)
            hip.synchronize()
            check(Y.values()[pick], t, xfmt, x, w, bias)
            assert Y.outside_kept()


@pytest.mark.parametrize("K", [100, 1100])
@pytest.mark.parametrize("M,N", SIZES)
def test_every_tile(gpu, M, N, K):
    every_output(M, N, K)


# rings of the tiles for few rows that turn more than once
@pytest.mark.parametrize("M,N", [(20, 65), (17, 3200), (3, 14000), (33, 5000), (20, 5000), (33, 6000), (40, 10001)])
def test_few_rows_of_many_stages(gpu, M, N):
    every_output(M, N, 4500)


class FarRows:
    """Rows of bytes `stride` apart in memory of which only they are written."""

    def __init__(self, rows, stride):
        self.stride, self.buf = stride, hip.DeviceBuffer(len(rows) * stride)
        for i, r in enumerate(np.ascontiguousarray(rows)):
            self.buf.upload(r, i * stride)
        self.ptr = self.buf.ptr


@pytest.mark.parametrize("M,N,stride", [(40, 1000, 5 << 20), (200, 1000, 5 << 20), (2050, 1000, 40 << 20), (1025, 7000, 1 << 20),
                                        (40, 120, 40 << 20)])
def test_rows_past_32_bits(gpu, M, N, stride):
    """W of 5 to 40 GB; the rows of one tile farther apart than 32 bits reach (40 << 20)."""
    K = 600
    wc, ws = random_rows(E2M1, N, K, 3)
    packed = np.zeros((N, tier_amd.mx_row_bytes(E2M1, K)), np.uint8)
    packed[:, :K // 2] = mx.pack(E2M1, wc)
    scales = np.zeros((N, tier_amd.mx_scale_bytes(K)), np.uint8)
    scales[:, :ws.shape[1]] = ws
    W, S, w = FarRows(packed, stride), FarRows(scales, 1 << 14), mx.values(E2M1, wc, ws)
    pick = some_rows(M, 4)
    for xfmt in (E2M1, E4M3):
        c, s = random_rows(xfmt, M, K, 5)
        X, Y = MxRows(xfmt, M, K, c, s), Rows(F32, M, N)
        tier_amd.mx_gemm(X.q.ptr, xfmt, X.rb, X.s.ptr, X.sb, W.ptr, stride, S.ptr, S.stride, None, Y.ptr, F32, N, M, N, K)
        hip.synchronize()
        check(Y.values()[pick], F32, xfmt, mx.values(xfmt, c[pick], s[pick]), w)


@pytest.mark.parametrize("M,N", [(1, 600), (2, 6000), (50, 400)])
def test_x_and_y_past_32_bits(gpu, M, N):
    """A linear whose weight, x and output all span more than 4 GiB."""
    K, far = 700, 3 << 30
    wc, ws = random_rows(E2M1, N, K, 6)
    packed = np.zeros((N, tier_amd.mx_row_bytes(E2M1, K)), np.uint8)
    packed[:, :K // 2] = mx.pack(E2M1, wc)
    scales = np.zeros((N, tier_amd.mx_scale_bytes(K)), np.uint8)
    scales[:, :ws.shape[1]] = ws
    W, S, w = FarRows(packed, 8 << 20), FarRows(scales, 1 << 12), mx.values(E2M1, wc, ws)
    x = np.random.default_rng(7).standard_normal((M, K)).astype(np.float32)
    rows = min(M, 50)
    stride = far if M <= 2 else 100 << 20
    X, Y = FarRows(x[:rows].view(np.uint8).reshape(rows, -1), stride), hip.DeviceBuffer(rows * stride)
    tier_amd.mx_linear(X.ptr, F32, stride // 4, E4M3, W.ptr, 8 << 20, S.ptr, 1 << 12, None, Y.ptr, F32, stride // 4, M, N, K)
    hip.synchronize()
    got = np.stack([Y.download(np.float32, N, i * stride) for i in range(M)]).astype(np.float64)
    c, s = mx.quantize(E4M3, x)
    check(got, F32, E4M3, mx.values(E4M3, c, s), w)
