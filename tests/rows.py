"""fp32 / fp16 / bf16 rows for the tests: host bits, device buffers with strides and odd starts."""
import collections

import numpy as np

import tier_amd
from tier_amd import hip

TYPES = (tier_amd.F32, tier_amd.F16, tier_amd.BF16)
#: unit roundoff of a type, and half its smallest subnormal
UNIT = {tier_amd.F32: 2.0 ** -24, tier_amd.F16: 2.0 ** -11, tier_amd.BF16: 2.0 ** -8}
TINY = {tier_amd.F32: 2.0 ** -150, tier_amd.F16: 2.0 ** -25, tier_amd.BF16: 2.0 ** -134}
SIZE = {tier_amd.F32: 4, tier_amd.F16: 2, tier_amd.BF16: 2}
_BITS = {tier_amd.F32: np.uint32, tier_amd.F16: np.uint16, tier_amd.BF16: np.uint16}


def to_bits(t, x):
    x = np.ascontiguousarray(x, np.float32)
    if t == tier_amd.F32:
        return x.view(np.uint32)
    if t == tier_amd.F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_bits(t, b):
    if t == tier_amd.F32:
        return b.view(np.float32)
    if t == tier_amd.F16:
        return b.view(np.float16).astype(np.float32)
    return (b.astype(np.uint32) << 16).view(np.float32)


class Rows:
    """rows x cols of type t on the device, `ld` elements apart, `skip` elements past an aligned
    start; what lies between rows holds a pattern that outside() compares."""

    def __init__(self, t, rows, cols, values=None, pad=0, skip=0):
        self.t, self.rows, self.cols, self.ld, self.skip = t, rows, cols, cols + pad, skip
        host = np.full(skip + rows * self.ld + 8, 0x3c3c if SIZE[t] == 2 else 0x3c3c3c3c, _BITS[t])
        if values is not None:
            bits = to_bits(t, values).reshape(rows, cols)
            for r in range(rows):
                host[skip + r * self.ld:skip + r * self.ld + cols] = bits[r]
        self.host = host
        self.buf = hip.to_device(host)
        self.ptr = self.buf.ptr + skip * SIZE[t]

    def _image(self):
        return self.buf.download(_BITS[self.t])

    def bits(self):
        img = self._image()[self.skip:self.skip + self.rows * self.ld]
        return img.reshape(self.rows, self.ld)[:, :self.cols] if self.rows else img.reshape(0, self.cols)

    def values(self):
        """What the rows hold now, as fp64."""
        return from_bits(self.t, np.ascontiguousarray(self.bits())).astype(np.float64)

    def outside_kept(self):
        now, was = self._image(), self.host.copy()
        for r in range(self.rows):
            s = slice(self.skip + r * self.ld, self.skip + r * self.ld + self.cols)
            now[s] = was[s] = 0
        return np.array_equal(now, was)


# calls take f32(...).ptr in place: the last tables made stay allocated while they run
_alive = collections.deque(maxlen=64)


def i32(a):
    _alive.append(hip.to_device(np.ascontiguousarray(a, np.int32)))
    return _alive[-1]


def f32(a):
    _alive.append(hip.to_device(np.ascontiguousarray(a, np.float32)))
    return _alive[-1]
