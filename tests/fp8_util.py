"""Matrices in 8-bit floating point for the tests: their codes in 64 bits, and device copies with marked gaps."""
from __future__ import annotations

import numpy as np

from gpu_util import Dev
from traincpp_amd import hip as H

BLOCK = 128


def _table():
    c = np.arange(128)
    e, m = c >> 3, (c & 7) / 8.0
    v = np.where(e > 0, (1 + m) * 2.0 ** (e - 7), m * 2.0 ** -6)
    v[127] = np.nan
    return np.concatenate([v, -v])


VALUES = _table()  # what each code stands for
_POSITIVE = VALUES[:127]
_MIDDLES = (_POSITIVE[1:] + _POSITIVE[:-1]) / 2


def encode(v):
    """The codes nearest to values of magnitude 448 at most (NaN: 0x7F), ties to even codes."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    lo = np.searchsorted(_MIDDLES, a, side="left")   # the lower neighbour on a tie
    hi = np.searchsorted(_MIDDLES, a, side="right")  # the upper one
    c = np.where(lo % 2 == 0, lo, hi)
    c = np.where(np.isnan(v), 127, np.minimum(c, 126)).astype(np.uint8)
    return np.where(np.signbit(v) & ~np.isnan(v), c | 128, c).astype(np.uint8)


def exponent(amax):
    """The exponent of a block's scale from its largest magnitudes."""
    amax = np.asarray(amax, np.float64)
    m, e = np.frexp(np.where(amax > 0, amax, 1.0))  # amax = m 2^e, 448 = 7/8 2^9
    e = np.maximum(e - 9 + (m > 0.875), -126)
    return np.where(amax > 0, e, 0)


def pad(x, rows, cols):
    out = np.zeros((-(-x.shape[0] // rows) * rows, -(-x.shape[1] // cols) * cols), x.dtype)
    out[:x.shape[0], :x.shape[1]] = x
    return out


def quantize(x, by_blocks=False):
    """x [R, K] in 64 bits: codes [R, blocks * 128] and exponents' bytes [R or blocks, blocks]."""
    R, K = x.shape
    finite = np.where(np.isfinite(x), x, 0.0)
    rows = BLOCK if by_blocks else 1
    p = pad(finite, rows, BLOCK)
    b = np.abs(p).reshape(p.shape[0] // rows, rows, -1, BLOCK).max((1, 3))
    e = exponent(b)
    s = np.repeat(np.repeat(2.0 ** e, rows, 0), BLOCK, 1)[:R]
    v = pad(np.where(np.isfinite(x), x, np.nan), 1, BLOCK) / s
    return encode(v), (e + 127).astype(np.uint8)


def values(codes, scales, K, by_blocks):
    """What codes [R, *] with scales (bytes or floats) stand for, [R, K]."""
    s = 2.0 ** (scales.astype(np.float64) - 127) if scales.dtype == np.uint8 else scales.astype(np.float64)
    s = np.repeat(s, BLOCK, 1)[:, :K]
    if by_blocks:
        s = np.repeat(s, BLOCK, 0)[:codes.shape[0]]
    return VALUES[codes[:, :K]] * s


class Bytes:
    """Rows of bytes or floats on the device, `pitch` bytes apart, from `lead` bytes after the allocation's start; what lies
    between them and around is marked, and read() checks that. `room`: bytes of a row that belong to it."""

    MARK = 0x5A

    def __init__(self, x, pitch, room, lead=0):
        self.x, self.pitch, self.room, self.lead = x, pitch, room, lead
        R = x.shape[0]
        raw = np.full(lead + R * pitch + 64, self.MARK, np.uint8)
        for r in range(R):
            row = np.zeros(room, np.uint8)
            b = np.ascontiguousarray(x[r]).view(np.uint8)
            row[:len(b)] = b
            raw[lead + r * pitch:lead + r * pitch + room] = row
        self.dev = Dev(raw)
        self.ptr = self.dev.ptr + lead

    def tensor(self, n, type_, es):
        R = self.x.shape[0]
        return H.tensor(self.ptr, [n, R, 1, 1], [es, self.pitch, self.pitch * R, self.pitch * R], type_)

    def read(self):
        """Every row's bytes, `room` of them."""
        raw = self.dev.read()
        R = self.x.shape[0]
        body = raw[self.lead:self.lead + R * self.pitch].reshape(R, self.pitch)
        assert np.all(raw[:self.lead] == self.MARK) and np.all(raw[self.lead + R * self.pitch:] == self.MARK)
        assert np.all(body[:, self.room:] == self.MARK), "bytes between rows were written"
        return body[:, :self.room].copy()

    def free(self):
        self.dev.free()


class Fp8:
    """A trc_hip_fp8 on the device. codes [R, K or more], scales [R or blocks, blocks]; `extra`: blocks between rows."""

    def __init__(self, codes, scales, K, extra=0, lead=0):
        R, kb = codes.shape[0], -(-K // BLOCK)
        room = kb * BLOCK
        c = np.zeros((R, room), np.uint8)
        c[:, :K] = codes[:, :K]
        self.codes, self.scales, self.K = c, scales, K
        self.q = Bytes(c, room + extra * BLOCK, room, lead * 16)
        es = scales.itemsize
        word = -(-kb * es // 4) * 4
        self.s = Bytes(scales, word + extra * 4, word, lead * 4)
        self.t = H.fp8(self.q.tensor(K, H.TYPE_I8, 1), self.s.tensor(kb, H.TYPE_I8 if es == 1 else H.TYPE_F32, es))

    def free(self):
        self.q.free()
        self.s.free()
