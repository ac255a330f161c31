"""What the entry points of adapter tuning refuse, before any device work: the addresses here
are never read, so the checks run without a GPU."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from conftest import ROOT
from traincpp_amd import hip as H

F32, F16, I32 = H.TYPE_F32, H.TYPE_F16, H.TYPE_I32


def tensor(at, *ne, type_=F32, nb=None):
    ne = list(ne) + [1] * (4 - len(ne))
    t = H.tensor(at << 32, ne, H.contiguous_nb(ne, 2 if type_ in (F16, H.TYPE_BF16) else 4), type_)
    for i, v in (nb or {}).items():
        t.nb[i] = v
    return t


def lora_args():
    """K 64, M 48, R 8, three adapters, five tokens, two requests; nothing overlaps."""
    return dict(a=tensor(1, 64, 8, 3), b=tensor(2, 8, 48, 3), scale=tensor(3, 3), start=tensor(4, 3, type_=I32),
                adapter=tensor(5, 2, type_=I32), x=tensor(6, 64, 5), h=tensor(7, 8, 5), base=tensor(8, 48, 5),
                dst=tensor(9, 48, 5), dy=tensor(10, 48, 5), g=tensor(11, 8, 5), dxb=tensor(12, 64, 5),
                dx=tensor(13, 64, 5), da=tensor(14, 64, 8, 3), db=tensor(15, 8, 48, 3))


def forward(q):
    H.lora(H.lora_set(q["a"], q["b"], q["scale"], q["start"], q["adapter"]), q["x"], q["base"], q["h"], q["dst"])


def backward(q):
    H.lora_back(H.lora_set(q["a"], q["b"], q["scale"], q["start"], q["adapter"]), q["x"], q["h"], q["dy"], q["g"],
                q["dxb"], q["dx"], q["da"], q["db"])


def refused(call, args, code):
    with pytest.raises(H.HipError) as e:
        call(args)
    assert e.value.code == code, str(e.value)


SHARED = [
    ("a", tensor(1, 64, 8, 3, type_=H.TYPE_Q4_0), H.E_INVALID),
    ("b", tensor(2, 8, 48, 3, type_=F16), H.E_INVALID),        # not a's type
    ("b", tensor(2, 9, 48, 3), H.E_SHAPE),
    ("b", tensor(2, 8, 48, 2), H.E_SHAPE),
    ("a", tensor(1, 64, 257, 3), H.E_SHAPE),
    ("a", tensor(1, 64, 0, 3), H.E_SHAPE),
    ("a", tensor(1, 64, 8, 0), H.E_SHAPE),
    ("a", tensor(1, 64, 8, 3, nb={0: 8}), H.E_ALIGN),          # strided along K
    ("a", tensor(1, 64, 8, 3, nb={1: 258}), H.E_ALIGN),
    ("scale", tensor(3, 2), H.E_SHAPE),
    ("start", tensor(4, 2, type_=I32), H.E_SHAPE),
    ("start", tensor(4, 3), H.E_INVALID),
    ("adapter", tensor(5, 0, type_=I32), H.E_SHAPE),
    ("adapter", tensor(5, 2, type_=I32, nb={0: 8}), H.E_ALIGN),
    ("x", tensor(6, 65, 5), H.E_SHAPE),
    ("x", tensor(6, 64, 0), H.E_SHAPE),
    ("x", tensor(6, 64, 5, type_=F16), H.E_INVALID),
    ("x", tensor(6, 64, 5, nb={0: 256, 1: 4}), H.E_ALIGN),
    ("x", tensor(0, 64, 5), H.E_ALIGN),
    ("h", tensor(7, 8, 5, nb={1: 64}), H.E_SHAPE),             # not contiguous
    ("h", tensor(7, 8, 4), H.E_SHAPE),
]


@pytest.mark.parametrize("name,value,code", SHARED)
def test_lora_and_its_gradients_refuse(name, value, code):
    for call in (forward, backward):
        refused(call, {**lora_args(), name: value}, code)


@pytest.mark.parametrize("name,value,code", [
    ("dst", tensor(9, 47, 5), H.E_SHAPE),
    ("dst", tensor(9, 48, 5, nb={1: 188}), H.E_SHAPE),         # rows overlap
    ("dst", tensor(6, 48, 5), H.E_SHAPE),                      # on x
    ("dst", tensor(2, 48, 5), H.E_SHAPE),                      # on the adapters
    ("dst", tensor(8, 48, 5, nb={1: 196}), H.E_SHAPE),         # on base, other rows
    ("h", tensor(6, 8, 5), H.E_SHAPE),
    ("base", tensor(8, 48, 4), H.E_SHAPE),
])
def test_lora_refuses(name, value, code):
    refused(forward, {**lora_args(), name: value}, code)


def test_lora_refuses_more_tiles_than_one_launch_holds():
    T = 6000000  # as many requests: a tile each, of 768 threads
    shapes = dict(a=tensor(1, 1, 1, 1), b=tensor(2, 1, 1, 1), scale=tensor(3, 1), start=tensor(4, T + 1, type_=I32),
                  adapter=tensor(5, T, type_=I32), x=tensor(6, 1, T), h=tensor(7, 1, T), base=tensor(8, 1, T), dst=tensor(9, 1, T))
    refused(forward, {**lora_args(), **shapes}, H.E_SHAPE)


def test_null_tensors():
    lib, q = H.load(), lora_args()
    s = H.lora_set(q["a"], q["b"], q["scale"], q["start"], q["adapter"])
    r = C.byref
    assert lib.trc_hip_lora(None, r(q["x"]), None, r(q["h"]), r(q["dst"]), None) == H.E_INVALID
    assert lib.trc_hip_lora(r(s), None, None, r(q["h"]), r(q["dst"]), None) == H.E_INVALID
    assert lib.trc_hip_lora(r(s), r(q["x"]), None, None, r(q["dst"]), None) == H.E_INVALID
    assert lib.trc_hip_lora(r(s), r(q["x"]), None, r(q["h"]), None, None) == H.E_INVALID
    for hole in range(8):
        args = [r(q[k]) for k in ("x", "h", "dy", "g", "dxb", "dx", "da", "db")]
        if hole == 4:
            continue  # base may be NULL
        args[hole] = None
        assert lib.trc_hip_lora_back(r(s), *args, 0, None) == H.E_INVALID, hole
    assert lib.trc_hip_preference_loss(None, None, None, None, 0.1, 0.0, None, None, None, None, None) == H.E_INVALID
    assert lib.trc_hip_adamw_create(None, 1, 32, r(C.c_void_p())) == H.E_INVALID
    assert lib.trc_hip_adamw_create(None, 0, 32, None) == H.E_INVALID
    assert lib.trc_hip_adamw_step(None, None, None) == H.E_INVALID
    assert lib.trc_hip_adamw_moments(None, None) == H.E_INVALID
    assert lib.trc_hip_adamw_destroy(None) == H.OK


@pytest.mark.parametrize("name,value,code", [
    ("dy", tensor(10, 47, 5), H.E_SHAPE),
    ("g", tensor(11, 8, 5, nb={1: 36}), H.E_SHAPE),
    ("dx", tensor(13, 65, 5), H.E_SHAPE),
    ("dx", None, H.E_INVALID),                                 # base without dx
    ("da", tensor(14, 64, 8, 2), H.E_SHAPE),
    ("da", tensor(14, 64, 8, 3, nb={2: 1024}), H.E_SHAPE),     # adapters overlap
    ("da", tensor(14, 64, 8, 3, type_=F16), H.E_INVALID),
    ("db", tensor(14, 8, 48, 3), H.E_SHAPE),                   # on da
    ("db", tensor(10, 8, 48, 3), H.E_SHAPE),                   # on dy
    ("g", tensor(7, 8, 5), H.E_SHAPE),                         # on h
    ("dx", tensor(6, 64, 5), H.E_SHAPE),                       # on x
])
def test_lora_back_refuses(name, value, code):
    refused(backward, {**lora_args(), name: value}, code)


def loss_args():
    """A vocabulary of 100, nine rows, two pairs."""
    return dict(logits=tensor(1, 100, 9), labels=tensor(2, 9, type_=I32), start=tensor(3, 5, type_=I32), ref=tensor(4, 4),
                beta=0.1, smoothing=0.0, lse=tensor(5, 9), logp=tensor(6, 4), slope=tensor(7, 2), loss=tensor(8, 1),
                dloss=tensor(9, 1), dlogits=tensor(10, 100, 9))


def loss(q):
    H.preference_loss(*(q[k] for k in ("logits", "labels", "start", "ref", "beta", "smoothing", "lse", "logp", "slope",
                                       "loss")))


def loss_back(q):
    H.preference_loss_back(*(q[k] for k in ("logits", "labels", "start", "lse", "slope", "dloss", "beta", "dlogits")))


@pytest.mark.parametrize("name,value,code", [
    ("logits", tensor(1, 100, 9, type_=I32), H.E_INVALID),
    ("logits", tensor(1, 100, 9, nb={0: 8}), H.E_ALIGN),
    ("logits", tensor(1, 0, 9), H.E_SHAPE),
    ("logits", tensor(1, 100, 9, 2), H.E_SHAPE),
    ("labels", tensor(2, 8, type_=I32), H.E_SHAPE),
    ("labels", tensor(2, 9), H.E_INVALID),
    ("start", tensor(3, 4, type_=I32), H.E_SHAPE),
    ("lse", tensor(5, 8), H.E_SHAPE),
    ("slope", tensor(7, 3), H.E_SHAPE),
    ("slope", tensor(7, 0), H.E_SHAPE),
    ("beta", float("nan"), H.E_INVALID),
])
def test_preference_loss_and_its_gradient_refuse(name, value, code):
    for call in (loss, loss_back):
        refused(call, {**loss_args(), name: value}, code)


@pytest.mark.parametrize("call,name,value,code", [
    (loss, "smoothing", -0.1, H.E_INVALID), (loss, "smoothing", 1.5, H.E_INVALID),
    (loss, "smoothing", float("nan"), H.E_INVALID), (loss, "ref", tensor(4, 3), H.E_SHAPE),
    (loss, "logp", tensor(5, 4), H.E_SHAPE), (loss, "loss", tensor(1, 1), H.E_SHAPE),
    (loss_back, "dlogits", tensor(10, 100, 8), H.E_SHAPE), (loss_back, "dlogits", tensor(10, 100, 9, type_=F16), H.E_INVALID),
    (loss_back, "dlogits", tensor(10, 100, 9, nb={1: 396}), H.E_SHAPE),
    (loss_back, "dlogits", tensor(1, 100, 9, nb={1: 404}), H.E_SHAPE),
    (loss_back, "dlogits", tensor(5, 100, 9), H.E_SHAPE), (loss_back, "dloss", tensor(9, 2), H.E_SHAPE),
])
def test_preference_refuses(call, name, value, code):
    refused(call, {**loss_args(), name: value}, code)


@pytest.mark.parametrize("V", [(1 << 30) + 1, (1 << 31) - 16384, (1 << 31) - 1, 1 << 31])
def test_preference_refuses_rows_that_32_bits_do_not_count(V):
    """Rows that lie on one another, as a stride of 0 has them, fit memory however long they are."""
    for call in (loss, loss_back):
        refused(call, {**loss_args(), "logits": tensor(1, V, 9, type_=F16, nb={1: 0}), "dlogits": tensor(99, V, 9, type_=F16)},
                H.E_SHAPE)


def plan(bits=32, **change):
    t = dict(param=1 << 32, grad=2 << 32, m=3 << 32, v=4 << 32, m_scale=5 << 32, v_scale=6 << 32, n=100)
    t.update(change)
    return H.AdamW([t], bits)


@pytest.mark.parametrize("bits,change,code", [
    (16, {}, H.E_INVALID), (32, {"n": -1}, H.E_SHAPE), (32, {"grad_type": H.TYPE_Q4_0}, H.E_INVALID),
    (32, {"param": 0}, H.E_ALIGN), (32, {"grad": (2 << 32) + 2}, H.E_ALIGN), (32, {"m": (3 << 32) + 1}, H.E_ALIGN),
    (8, {"m_scale": 0}, H.E_ALIGN), (8, {"v_scale": (6 << 32) + 2}, H.E_ALIGN), (32, {"v_out": 3}, H.E_ALIGN),
    (8, {"v": 0}, H.E_ALIGN), (32, {"n": 1 << 40}, H.E_SHAPE),
])
def test_adamw_refuses(bits, change, code):
    with pytest.raises(H.HipError) as e:
        plan(bits, **change)
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [(1 << 24) * 2048, (1 << 62), (1 << 63) - 2048, (1 << 63) - 1])
def test_adamw_refuses_tensors_up_to_the_largest_size(bits, n):
    """... the last of which overflow 64 bits if they are rounded up before they are divided."""
    with pytest.raises(H.HipError) as e:
        plan(bits, n=n)
    assert e.value.code == H.E_SHAPE and "elements in one plan" in str(e.value), str(e.value)


@pytest.mark.parametrize("entry,call", [
    ("trc_hip_lora", "R.forward(R.lora_args())"), ("trc_hip_lora_back", "R.backward(R.lora_args())"),
    ("trc_hip_preference_loss", "R.loss(R.loss_args())"), ("trc_hip_preference_loss_back", "R.loss_back(R.loss_args())"),
    ("trc_hip_adamw_create", "R.plan()"),
])
def test_forced_errors(entry, call):
    code = f"import conftest\nimport test_tuning_refusals as R\ntry:\n    {call}\nexcept R.H.HipError as e:\n    print(e.code)\n"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=str(ROOT / "tests"), timeout=120,
                       env={**os.environ, "TRC_HIP_FORCE_ERROR": entry})
    assert r.returncode == 0 and r.stdout.strip() == "-5", r.stdout + r.stderr


def test_tensors_outside_of_hip_buffers_abort():
    r = subprocess.run([str(ROOT / "tests" / "cpp" / "bin" / "test_tuning"), "--abort-host"], capture_output=True, text=True,
                       timeout=60)
    assert r.returncode != 0
    assert "not in a HIP buffer" in r.stderr
