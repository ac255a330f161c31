"""Calls of the 8-bit products and the distillation loss that stand apart: rows whose offsets pass 32 bits, two streams at
once, and the operators one after another on one stream's workspace. Each is held to the bits of the same call on
compact tensors, alone (whose values the other files' tests hold to 64 bits)."""
import numpy as np
import pytest

import fp8_util as F
from conftest import announce
from gpu_util import Stream
from traincpp_amd import hip as H
from tuning_util import TYPES, Mat, vec

pytestmark = pytest.mark.gpu


class Far:
    """A matrix whose rows lie `pitch` bytes apart."""

    def __init__(self, x, pitch, kind, room=None):
        self.x, self.pitch = x, pitch
        self.room = room or x.shape[1] * x.itemsize
        self.buf = H.DeviceBuffer(pitch * (len(x) - 1) + self.room)
        for r, row in enumerate(x):
            raw = np.zeros(self.room, np.uint8)
            raw[:row.nbytes] = np.ascontiguousarray(row).view(np.uint8)
            H.check(H.load().trc_hip_h2d(self.buf.ptr + r * pitch, raw.ctypes.data, self.room, None))
        R, n = x.shape
        self.t = H.tensor(self.buf.ptr, [n, R, 1, 1], [x.itemsize, pitch, pitch * R, pitch * R], kind)

    def read(self):
        out = np.empty_like(self.x)
        for r in range(len(out)):
            row = np.empty_like(out[r])
            H.check(H.load().trc_hip_d2h(row.ctypes.data, self.buf.ptr + r * self.pitch, row.nbytes, None))
            out[r] = row
        return out

    def free(self):
        self.buf.free()


def far8(codes, scales, K, pitch, spitch):
    kb = -(-K // 128)
    q = Far(np.ascontiguousarray(codes[:, :K]), pitch, H.TYPE_I8, kb * 128)
    s = Far(np.ascontiguousarray(scales), spitch, H.TYPE_I8 if scales.itemsize == 1 else H.TYPE_F32,
            -(-kb * scales.itemsize // 4) * 4)
    return H.fp8(q.t, s.t), q, s


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("N", [40, 600])
def test_offsets_past_32_bits(hip, kind, N):
    """Codes 8 MiB from row to row, scales 4 MiB, results and inputs 16 MiB."""
    announce(f"fp8 far rows {kind} N={N}")
    K, M, MIB = 300, 290, 1 << 20
    rng = np.random.default_rng(N)
    dt = {"f32": np.float32, "bf16": np.uint16}[kind]
    w, ws = F.quantize(rng.standard_normal((M, K)), True)
    xv = rng.standard_normal((N, K)).astype(np.float32)
    g, gs = F.quantize(rng.standard_normal((N, M)))
    near = F.Fp8(w, ws, K)
    xq = F.Fp8(np.zeros((N, K), np.uint8), np.zeros((N, 3), np.uint8), K)
    gq = F.Fp8(g, gs, M)
    x, y, dx = Mat(xv), Mat(np.zeros((N, M), dt), TYPES[kind]), Mat(np.zeros((N, K), dt), TYPES[kind])
    H.fp8_quantize(x.t, xq.t)
    H.fp8_mul_mat(near.t, xq.t, y.t)
    H.fp8_mul_mat_back(near.t, gq.t, dx.t)
    H.sync()
    fw, *b1 = far8(w, ws, K, 8 * MIB, 4 * MIB)
    fx, *b2 = far8(np.zeros((N, K), np.uint8), np.zeros((N, 3), np.uint8), K, 8 * MIB, 4 * MIB)
    fg, *b3 = far8(g, gs, M, 8 * MIB, 4 * MIB)
    fxv, fy, fdx = Far(xv, 16 * MIB, H.TYPE_F32), Far(np.zeros((N, M), dt), 16 * MIB, TYPES[kind]), Far(np.zeros((N, K), dt), 16 * MIB, TYPES[kind])
    H.fp8_quantize(fxv.t, fx)
    H.fp8_mul_mat(fw, fx, fy.t)
    H.fp8_mul_mat_back(fw, fg, fdx.t)
    H.sync()
    assert np.array_equal(b2[0].read(), xq.q.read()[:, :K])
    assert np.array_equal(fy.read(), y.read()) and np.array_equal(fdx.read(), dx.read())
    if N <= H.FP8_MATVEC_MAX_N:
        H.fp8_matvec(fw, fxv.t, cleared(fy).t)
        H.sync()
        assert np.array_equal(fy.read(), y.read())
    for b in (near, xq, gq, x, y, dx, fxv, fy, fdx, *b1, *b2, *b3):
        b.free()


def cleared(m):
    """The same matrix, cleared."""
    for r in range(len(m.x)):
        raw = np.zeros(m.room, np.uint8)
        H.check(H.load().trc_hip_h2d(m.buf.ptr + r * m.pitch, raw.ctypes.data, m.room, None))
    return m


class Distill:
    def __init__(self, seed, V=40000, T=11, top=30, kind=np.float32):
        rng = np.random.default_rng(seed)
        self.l = rng.standard_normal((T, V)).astype(kind)
        self.ids = rng.integers(0, V, (T, top)).astype(np.int32)
        self.z = rng.standard_normal((T, top)).astype(np.float32)
        self.y = rng.integers(-1, V, T).astype(np.int32)
        self.T, self.V = T, V

    def place(self, logits, d):
        self.lt, self.dt = logits, d
        self.ids_d, self.z_d, self.stats = Mat(self.ids, H.TYPE_I32), Mat(self.z), Mat(np.zeros((self.T, 5), np.float32))
        self.y_d, self.yt = vec(self.y, H.TYPE_I32)
        self.loss, self.loss_t = vec(np.zeros(4, np.float32), H.TYPE_F32)
        self.one, self.one_t = vec(np.ones(1, np.float32), H.TYPE_F32)

    def run(self, s=None):
        H.distill_loss(self.lt.t, self.yt, self.ids_d.t, self.z_d.t, 2.0, 0.7, self.stats.t, self.loss_t, s)
        H.distill_loss_back(self.lt.t, self.yt, self.ids_d.t, self.z_d.t, self.stats.t, self.loss_t, self.one_t, 2.0, 0.7, self.dt.t, s)

    def free(self):
        for b in (self.lt, self.dt, self.ids_d, self.z_d, self.stats, self.y_d, self.loss, self.one):
            b.free()


def test_distillation_of_far_rows(hip):
    announce("distill far rows")
    p, q = Distill(3, V=9001, T=300), Distill(3, V=9001, T=300)
    p.place(Mat(p.l), Mat(np.zeros_like(p.l)))
    q.place(Far(q.l, 16 << 20, H.TYPE_F32), Far(np.zeros_like(q.l), 16 << 20, H.TYPE_F32))
    p.run()
    q.run()
    H.sync()
    assert np.array_equal(p.loss.read(), q.loss.read()) and np.array_equal(p.dt.read(), q.dt.read())
    p.free()
    q.free()


class Step:
    """A few tokens with sums in parts, the single-token form by way of the workspace, and a loss of rows in parts."""

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        K, M, N = 4000, 500, 100
        self.w = F.Fp8(*F.quantize(rng.standard_normal((M, K)), True), K)
        self.x = Mat(rng.standard_normal((N, K)).astype(np.float32))
        self.few = Mat(rng.standard_normal((7, K)).astype(np.float32))
        self.xq = F.Fp8(np.zeros((N, K), np.uint8), np.zeros((N, 32), np.uint8), K)
        self.y, self.yf = Mat(np.zeros((N, M), np.float32)), Mat(np.zeros((7, M), np.float32))
        self.d = Distill(seed)
        self.d.place(Mat(self.d.l), Mat(np.zeros_like(self.d.l)))

    def run(self, s=None):
        H.fp8_quantize(self.x.t, self.xq.t, s)
        H.fp8_mul_mat(self.w.t, self.xq.t, self.y.t, s)
        H.fp8_matvec(self.w.t, self.few.t, self.yf.t, s)
        self.d.run(s)

    def read(self):
        return [self.y.read(), self.yf.read(), self.d.loss.read(), self.d.dt.read()]

    def free(self):
        for b in (self.w, self.x, self.few, self.xq, self.y, self.yf, self.d):
            b.free()


def test_two_streams_at_once(hip):
    announce("fp8 and distill on two streams")
    steps = [Step(5), Step(6)]
    want = []
    for p in steps:
        p.run()
        H.sync()
        want.append(p.read())
    streams = [Stream(), Stream()]
    for p, s in zip(steps, streams):
        p.run(s.handle)
    for _ in range(20):
        for p, s in zip(steps, streams):
            p.run(s.handle)
    for s in streams:
        H.sync(s.handle)
    for p, w in zip(steps, want):
        for a, b in zip(p.read(), w):
            assert np.array_equal(a, b)
        p.free()
    for s in streams:
        s.close()
