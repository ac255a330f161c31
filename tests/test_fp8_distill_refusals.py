"""What the 8-bit products and the distillation loss refuse, before any device work: the addresses here are never read,
so the checks run without a GPU."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT
from traincpp_amd import hip as H

F32, F16, BF16, I8, I32 = H.TYPE_F32, H.TYPE_F16, H.TYPE_BF16, H.TYPE_I8, H.TYPE_I32
SIZE = {F32: 4, F16: 2, BF16: 2, I8: 1, I32: 4}


def tensor(at, *ne, type_=F32, nb=None, off=0):
    ne = list(ne) + [1] * (4 - len(ne))
    t = H.tensor((at << 36) + off if at else 0, ne, H.contiguous_nb(ne, SIZE.get(type_, 4)), type_)
    for i, v in (nb or {}).items():
        t.nb[i] = v
    return t


def codes(at, K, R, pitch=None, **kw):
    pitch = -(-K // 128) * 128 if pitch is None else pitch
    return tensor(at, K, R, type_=I8, nb={1: pitch, 2: pitch * R, 3: pitch * R}, **kw)


def bytes_(at, K, R, pitch=None, **kw):
    kb = -(-K // 128)
    pitch = -(-kb // 4) * 4 if pitch is None else pitch
    return tensor(at, kb, R, type_=I8, nb={1: pitch, 2: pitch * R, 3: pitch * R}, **kw)


def args():
    """K 300, M 200, 70 tokens; nothing overlaps."""
    return dict(wq=codes(1, 300, 200), ws=tensor(2, 3, 2), xq=codes(3, 300, 70), xs=bytes_(4, 300, 70), y=tensor(5, 200, 70),
                gq=codes(6, 200, 70), gs=bytes_(7, 200, 70), dx=tensor(8, 300, 70, type_=BF16), x=tensor(9, 300, 70),
                x1=tensor(10, 300, 9, type_=F16), y1=tensor(11, 200, 9))


def product(q):
    H.fp8_mul_mat(H.fp8(q["wq"], q["ws"]), H.fp8(q["xq"], q["xs"]), q["y"])


def back(q):
    H.fp8_mul_mat_back(H.fp8(q["wq"], q["ws"]), H.fp8(q["gq"], q["gs"]), q["dx"])


def matvec(q):
    H.fp8_matvec(H.fp8(q["wq"], q["ws"]), q["x1"], q["y1"])


def quantize(q):
    H.fp8_quantize(q["x"], H.fp8(q["xq"], q["xs"]))


def refused(call, args, code):
    with pytest.raises(H.HipError) as e:
        call(args)
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("name,value,code", [
    ("wq", codes(1, 300, 200, off=8), H.E_ALIGN),
    ("wq", codes(1, 300, 200, pitch=320), H.E_ALIGN),
    ("wq", codes(1, 300, 200, pitch=256), H.E_SHAPE),          # no room for whole blocks
    ("wq", codes(1, 300, 200, pitch=(1 << 23) + 128), H.E_SHAPE),
    ("wq", tensor(1, 300, 200, type_=F16), H.E_INVALID),
    ("wq", codes(0, 300, 200), H.E_ALIGN),
    ("wq", codes(1, 0, 200, pitch=384), H.E_SHAPE),
    ("wq", codes(1, (1 << 23) + 1, 200), H.E_SHAPE),
    ("ws", tensor(2, 2, 2), H.E_SHAPE),
    ("ws", tensor(2, 3, 200), H.E_SHAPE),                      # a weight has no scales of its rows
    ("ws", tensor(2, 3, 2, type_=F16), H.E_INVALID),
    ("ws", tensor(2, 3, 2, type_=I8), H.E_ALIGN),              # rows of three bytes
    ("ws", bytes_(2, 300, 2, off=2), H.E_ALIGN),
    ("ws", tensor(2, 3, 2, nb={0: 8}), H.E_ALIGN),
    ("ws", tensor(0, 3, 2), H.E_ALIGN),
])
def test_products_refuse_a_weight(name, value, code):
    for call in (product, back, matvec):
        refused(call, {**args(), name: value}, code)


@pytest.mark.parametrize("call,name,value,code", [
    (product, "xq", codes(3, 301, 70), H.E_SHAPE), (product, "xq", codes(3, 300, 69), H.E_SHAPE),
    (product, "xs", tensor(4, 3, 70), H.E_INVALID), (product, "xs", bytes_(4, 300, 1), H.E_SHAPE),
    (product, "xs", bytes_(4, 300, 70, pitch=6), H.E_ALIGN), (product, "xs", bytes_(4, 300, 70, pitch=(1 << 22) + 4), H.E_SHAPE),
    (product, "y", tensor(5, 300, 70), H.E_SHAPE), (product, "y", tensor(5, 200, 70, type_=I32), H.E_INVALID),
    (product, "y", tensor(5, 200, 70, nb={1: 796}), H.E_SHAPE), (product, "y", tensor(5, 200, 70, nb={0: 8}), H.E_ALIGN),
    (product, "y", tensor(5, 200, 70, off=2), H.E_ALIGN),
    (product, "y", tensor(1, 200, 70), H.E_SHAPE), (product, "y", tensor(2, 200, 70), H.E_SHAPE),
    (product, "y", tensor(3, 200, 70), H.E_SHAPE), (product, "y", tensor(4, 200, 70), H.E_SHAPE),
    (product, "y", tensor(3, 200, 70, off=69 * 384 + 380), H.E_SHAPE),  # in the last block's room
    (back, "gq", codes(6, 300, 70), H.E_SHAPE), (back, "gs", bytes_(7, 384 + 1, 70), H.E_SHAPE),
    (back, "dx", tensor(8, 200, 70), H.E_SHAPE), (back, "dx", tensor(6, 300, 70), H.E_SHAPE),
    (matvec, "x1", tensor(10, 300, 65), H.E_SHAPE), (matvec, "x1", tensor(10, 300, 0), H.E_SHAPE),
    (matvec, "x1", tensor(10, 299, 9), H.E_SHAPE), (matvec, "x1", tensor(10, 300, 9, type_=I8), H.E_INVALID),
    (matvec, "y1", tensor(11, 200, 8), H.E_SHAPE), (matvec, "y1", tensor(10, 200, 9), H.E_SHAPE),
    (quantize, "x", tensor(9, 299, 70), H.E_SHAPE), (quantize, "x", tensor(9, 300, 70, type_=I8), H.E_INVALID),
    (quantize, "x", tensor(9, 300, 70, nb={0: 8}), H.E_ALIGN), (quantize, "x", tensor(3, 300, 70), H.E_SHAPE),
    (quantize, "x", tensor(4, 300, 70), H.E_SHAPE), (quantize, "xs", tensor(4, 3, 1), H.E_INVALID),  # scales made are bytes
    (quantize, "xs", bytes_(3, 300, 70), H.E_SHAPE), (quantize, "xs", bytes_(4, 300, 2), H.E_SHAPE),
])
def test_products_refuse(call, name, value, code):
    refused(call, {**args(), name: value}, code)


def test_sizes_past_a_launch():
    """More blocks or tiles than one launch holds; rows that lie on one another fit memory however many they are."""
    big = 1 << 23
    x = tensor(1, big, big, type_=BF16, nb={1: 0})
    q = H.fp8(codes(2, big, big), bytes_(300, big, big >> 7))
    refused(lambda a: H.fp8_quantize(x, q), {}, H.E_SHAPE)
    w = H.fp8(codes(2, 128, big), bytes_(400, 128, big >> 7))
    y = tensor(500, big, big, type_=BF16)
    refused(lambda a: H.fp8_mul_mat(w, H.fp8(codes(600, 128, big), bytes_(700, 128, big)), y), {}, H.E_SHAPE)


def test_null_arguments():
    lib, q = H.load(), args()
    import ctypes as C
    r, w = C.byref, H.fp8(q["wq"], q["ws"])
    x = H.fp8(q["xq"], q["xs"])
    for f in (lib.trc_hip_fp8_mul_mat, lib.trc_hip_fp8_mul_mat_back):
        assert f(None, r(x), r(q["y"]), None) == H.E_INVALID
        assert f(r(w), None, r(q["y"]), None) == H.E_INVALID
        assert f(r(w), r(x), None, None) == H.E_INVALID
    assert lib.trc_hip_fp8_matvec(None, r(q["x1"]), r(q["y1"]), None) == H.E_INVALID
    assert lib.trc_hip_fp8_matvec(r(w), None, r(q["y1"]), None) == H.E_INVALID
    assert lib.trc_hip_fp8_matvec(r(w), r(q["x1"]), None, None) == H.E_INVALID
    assert lib.trc_hip_fp8_quantize(None, r(x), None) == H.E_INVALID
    assert lib.trc_hip_fp8_quantize(r(q["x"]), None, None) == H.E_INVALID
    t = loss_args()
    names = ("logits", "labels", "ids", "teacher", "stats", "loss")
    for hole in names:
        a = [None if k == hole else r(t[k]) for k in names]
        assert lib.trc_hip_distill_loss(*a[:4], 2.0, 0.5, *a[4:], None) == H.E_INVALID, hole
        assert lib.trc_hip_distill_loss_back(*a, r(t["dloss"]), 2.0, 0.5, r(t["dlogits"]), None) == H.E_INVALID, hole
    a = [r(t[k]) for k in names]
    assert lib.trc_hip_distill_loss_back(*a, None, 2.0, 0.5, r(t["dlogits"]), None) == H.E_INVALID
    assert lib.trc_hip_distill_loss_back(*a, r(t["dloss"]), 2.0, 0.5, None, None) == H.E_INVALID


# ------------------------------------------------------------------ distillation

def loss_args():
    """A vocabulary of 100, nine rows, four entries."""
    return dict(logits=tensor(1, 100, 9), labels=tensor(2, 9, type_=I32), ids=tensor(3, 4, 9, type_=I32),
                teacher=tensor(4, 4, 9, type_=BF16), tau=2.0, alpha=0.5, stats=tensor(5, 5, 9), loss=tensor(6, 4),
                dloss=tensor(7, 1), dlogits=tensor(8, 100, 9))


def loss(q):
    H.distill_loss(*(q[k] for k in ("logits", "labels", "ids", "teacher", "tau", "alpha", "stats", "loss")))


def loss_back(q):
    H.distill_loss_back(*(q[k] for k in ("logits", "labels", "ids", "teacher", "stats", "loss", "dloss", "tau", "alpha", "dlogits")))


@pytest.mark.parametrize("name,value,code", [
    ("logits", tensor(1, 100, 9, type_=I32), H.E_INVALID), ("logits", tensor(1, 100, 9, nb={0: 8}), H.E_ALIGN),
    ("logits", tensor(1, 0, 9), H.E_SHAPE), ("logits", tensor(1, 100, 9, 2), H.E_SHAPE),
    ("logits", tensor(1, (1 << 30) + 1, 9, type_=F16, nb={1: 0}), H.E_SHAPE),
    ("labels", tensor(2, 8, type_=I32), H.E_SHAPE), ("labels", tensor(2, 9), H.E_INVALID),
    ("ids", tensor(3, 4, 8, type_=I32), H.E_SHAPE), ("ids", tensor(3, 4, 9), H.E_INVALID),
    ("ids", tensor(3, 4, 9, type_=I32, nb={1: 20}), H.E_SHAPE), ("ids", tensor(3, 1025, 9, type_=I32), H.E_SHAPE),
    ("ids", tensor(3, 0, 9, type_=I32), H.E_SHAPE),
    ("teacher", tensor(4, 5, 9, type_=BF16), H.E_SHAPE), ("teacher", tensor(4, 4, 9, type_=I32), H.E_INVALID),
    ("teacher", tensor(4, 4, 9, nb={1: 20}), H.E_SHAPE),
    ("stats", tensor(5, 4, 9), H.E_SHAPE), ("stats", tensor(5, 5, 9, nb={1: 24}), H.E_SHAPE), ("loss", tensor(6, 1), H.E_SHAPE),
    ("tau", 0.0, H.E_INVALID), ("tau", -1.0, H.E_INVALID), ("tau", float("nan"), H.E_INVALID), ("tau", float("inf"), H.E_INVALID),
    ("tau", 1e-45, H.E_INVALID), ("alpha", -0.1, H.E_INVALID), ("alpha", 1.5, H.E_INVALID), ("alpha", float("nan"), H.E_INVALID),
])
def test_distill_loss_and_its_gradient_refuse(name, value, code):
    for call in (loss, loss_back):
        refused(call, {**loss_args(), name: value}, code)


@pytest.mark.parametrize("call,name,value,code", [
    (loss, "stats", tensor(1, 5, 9), H.E_SHAPE), (loss, "loss", tensor(5, 4), H.E_SHAPE), (loss, "loss", tensor(4, 4), H.E_SHAPE),
    (loss_back, "dlogits", tensor(8, 100, 8), H.E_SHAPE), (loss_back, "dlogits", tensor(8, 100, 9, type_=F16), H.E_INVALID),
    (loss_back, "dlogits", tensor(8, 100, 9, nb={1: 396}), H.E_SHAPE), (loss_back, "dlogits", tensor(1, 100, 9, nb={1: 404}), H.E_SHAPE),
    (loss_back, "dlogits", tensor(5, 100, 9), H.E_SHAPE), (loss_back, "dlogits", tensor(3, 100, 9), H.E_SHAPE),
    (loss_back, "dloss", tensor(7, 2), H.E_SHAPE),
])
def test_distill_refuses(call, name, value, code):
    refused(call, {**loss_args(), name: value}, code)


def test_more_rows_than_the_workspace_holds():
    T = (1 << 19) + 1
    q = dict(logits=tensor(1, 100, T), labels=tensor(2, T, type_=I32), ids=tensor(3, 4, T, type_=I32), teacher=tensor(4, 4, T),
             stats=tensor(5, 5, T), dlogits=tensor(8, 100, T))
    for call in (loss, loss_back):
        refused(call, {**loss_args(), **q}, H.E_SHAPE)


@pytest.mark.parametrize("entry,call", [
    ("trc_hip_fp8_quantize", "R.quantize(R.args())"), ("trc_hip_fp8_mul_mat", "R.product(R.args())"),
    ("trc_hip_fp8_mul_mat_back", "R.back(R.args())"), ("trc_hip_fp8_matvec", "R.matvec(R.args())"),
    ("trc_hip_distill_loss", "R.loss(R.loss_args())"), ("trc_hip_distill_loss_back", "R.loss_back(R.loss_args())"),
])
def test_forced_errors(entry, call):
    code = f"import conftest\nimport test_fp8_distill_refusals as R\ntry:\n    {call}\nexcept R.H.HipError as e:\n    print(e.code)\n"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=str(ROOT / "tests"), timeout=120,
                       env={**os.environ, "TRC_HIP_FORCE_ERROR": entry})
    assert r.returncode == 0 and r.stdout.strip() == "-5", r.stdout + r.stderr


def test_tensors_outside_of_hip_buffers_abort():
    r = subprocess.run([str(ROOT / "tests" / "cpp" / "bin" / "test_distillation"), "--abort-host"], capture_output=True, text=True,
                       timeout=60)
    assert r.returncode != 0
    assert "not in a HIP buffer" in r.stderr
