"""Microscaled rows for the tests, from the formats' definition: numbers, codes, device rows with strides."""
import numpy as np

import tier_amd
from tier_amd import hip

E2M1, E4M3 = tier_amd.MX_E2M1, tier_amd.MX_E4M3
FORMATS = (E2M1, E4M3)
#: the numbers of the codes without a sign, in order (E4M3's 0x7f is NaN)
LEVELS = {E2M1: np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6]),
          E4M3: np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
                          for e in range(16) for m in range(8)][:127])}
EMAX = {E2M1: 2, E4M3: 8}


def numbers(fmt, codes):
    """The numbers that codes stand for, under a scale of 1."""
    sign = 1 << (fmt - 1)
    return np.where(codes & sign, -1.0, 1.0) * LEVELS[fmt][codes & (sign - 1)]


def nearest(fmt, v):
    """Codes of the nearest numbers, ties to the even code, the largest for what is past it."""
    lv = LEVELS[fmt]
    a = np.minimum(np.abs(v), lv[-1])
    hi = np.minimum(np.searchsorted(lv, a), len(lv) - 1)
    lo = np.maximum(hi - 1, 0)
    down, up = a - lv[lo], lv[hi] - a
    c = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return c + np.where(np.signbit(v), 1 << (fmt - 1), 0)


def quantize(fmt, x):
    """(codes [M][K], scale bytes [M][blocks]) of fp32 rows by the definition in the header."""
    x = np.asarray(x, np.float32).astype(np.float64)
    M, K = x.shape
    b = np.zeros((M, -(-K // 32), 32))
    b.reshape(M, -1)[:, :K] = x
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 0, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    byte = np.where(top > 0, np.clip(np.frexp(top)[1] - 1 - EMAX[fmt] + 127, 0, 254), 0)
    codes = nearest(fmt, np.where(bad[..., None], 0, b) * np.exp2(127.0 - byte)[..., None])
    codes = np.where(bad[..., None], 0, codes)
    return codes.reshape(M, -1)[:, :K].astype(np.int64), np.where(bad, 255, byte).astype(np.int64)


def values(fmt, codes, scales):
    """fp64 rows; NaN under the scale 255."""
    K = codes.shape[1]
    s = np.where(scales == 255, np.nan, np.exp2(scales - 127.0))
    return numbers(fmt, codes) * np.repeat(s, 32, 1)[:, :K]


def pack(fmt, codes):
    """Bytes of a row's codes."""
    if fmt == E4M3:
        return codes.astype(np.uint8)
    c = np.zeros((codes.shape[0], -(-codes.shape[1] // 2) * 2), np.uint8)
    c[:, :codes.shape[1]] = codes
    return c[:, 0::2] | (c[:, 1::2] << 4)


def unpack(fmt, rows, K):
    if fmt == E4M3:
        return rows[:, :K].astype(np.int64)
    return np.stack([rows & 15, rows >> 4], -1).reshape(rows.shape[0], -1)[:, :K].astype(np.int64)


class MxRows:
    """Device rows of codes and their scales, `pad` 16-byte units further apart than they need be, with
    0x55 between them."""

    def __init__(self, fmt, rows, K, codes=None, scales=None, pad=0):
        self.fmt, self.rows, self.K = fmt, rows, K
        self.need, self.need_s = tier_amd.mx_row_bytes(fmt, K), tier_amd.mx_scale_bytes(K)
        self.rb, self.sb = self.need + 16 * pad, self.need_s + 16 * pad
        h = np.full((rows, self.rb), 0x55, np.uint8)
        s = np.full((rows, self.sb), 0x55, np.uint8)
        if codes is not None:
            h[:, :self.need] = 0
            s[:, :self.need_s] = 0
            p = pack(fmt, codes)
            h[:, :p.shape[1]] = p
            s[:, :scales.shape[1]] = scales
        self.q, self.s = hip.to_device(h), hip.to_device(s)

    def get(self):
        """(codes, scales of whole blocks) as they are now; checks the padding and what lies between rows."""
        h = self.q.download(np.uint8).reshape(self.rows, self.rb)
        s = self.s.download(np.uint8).reshape(self.rows, self.sb)
        used, blocks = -(-self.K * self.fmt // 8), -(-self.K // 32)
        assert not h[:, used:self.need].any() and not s[:, blocks:self.need_s].any(), "padding"
        assert (h[:, self.need:] == 0x55).all() and (s[:, self.need_s:] == 0x55).all(), "between rows"
        return unpack(self.fmt, h, self.K), s[:, :blocks].astype(np.int64)
