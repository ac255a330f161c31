"""Inputs and device views shared by the tests of adapters, preference loss and AdamW."""
from __future__ import annotations

import numpy as np

from gpu_util import Dev
from traincpp_amd import hip as H

TYPES = {"f32": H.TYPE_F32, "f16": H.TYPE_F16, "bf16": H.TYPE_BF16}
U32 = 2.0 ** -24  # rounding to 32 bits, relative


def to_bf16(x):
    """bf16 bits of float values, to nearest even (no NaNs)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def encode(x, kind):
    """x as `kind`, and the values that it then stands for in 64 bits."""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x, x.astype(np.float64)
    if kind == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float64)
    h = to_bf16(x)
    return h, decode(h, kind)


def decode(x, kind):
    if kind == "bf16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def rows(x, pad=0, lead=0):
    """A buffer that holds the matrix x with `pad` elements after each row, `lead` before
    the first and one more row, all of it filled with a mark; and the view of x in it."""
    r, c = x.shape
    mark = {2: 0x5A5A, 4: 0x5A5A5A5A}[x.dtype.itemsize]
    base = np.full(lead + (r + 1) * (c + pad), mark, {2: np.uint16, 4: np.uint32}[x.dtype.itemsize]).view(x.dtype)
    view = base[lead:lead + r * (c + pad)].reshape(r, c + pad)[:, :c]
    view[...] = x
    return base, view


class Mat:
    """A matrix on the device with gaps around its rows; read() checks the gaps."""

    def __init__(self, x, kind=H.TYPE_F32, pad=0, lead=0):
        self.shape, self.pad, self.lead = x.shape, pad, lead
        base, view = rows(x, pad, lead)
        self.dev = Dev(base)
        off = view.__array_interface__["data"][0] - base.__array_interface__["data"][0]
        es = x.dtype.itemsize
        r, c = x.shape
        nb1 = es * (c + pad)
        self.t = H.tensor(self.dev.ptr + off, [c, r, 1, 1], [es, nb1, nb1 * r, nb1 * r], kind)

    def read(self):
        base = self.dev.read()
        r, c = self.shape
        view = base[self.lead:self.lead + r * (c + self.pad)].reshape(r, c + self.pad)[:, :c]
        got = view.copy()
        ints = base.view({2: np.uint16, 4: np.uint32}[base.itemsize])
        keep = np.ones(base.shape, bool)
        keep[self.lead:self.lead + r * (c + self.pad)].reshape(r, c + self.pad)[:, :c] = False
        mark = {2: 0x5A5A, 4: 0x5A5A5A5A}[base.itemsize]
        assert np.all(ints[keep] == mark), "bytes outside the matrix were written"
        return got

    def free(self):
        self.dev.free()


def vec(x, kind):
    """A contiguous vector on the device and its descriptor."""
    d = Dev(x)
    es = x.dtype.itemsize
    return d, H.tensor(d.ptr, [x.size, 1, 1, 1], [es] + [es * x.size] * 3, kind)


def starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
