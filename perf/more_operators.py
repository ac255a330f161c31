"""The operators of distillation beside an 8-bit weight as cases to be timed and checked.

A case is a dict of plain values; its "op" says what a pass is:

  fp8        a projection whose weight is held in 8-bit floating point (e4m3) with a
             scale for each block of 128 x 128: the activations are quantized, each
             token's in blocks of 128 with a power of two for scale, and multiplied:
             y = W q(x)
  fp8_back   the gradient by its activations, the incoming one quantized the same way
             along the weight's rows: dx = W^T q(dy)
  distill    the loss of a student's logits against a teacher's top logits, mixed with
             the labels' cross-entropy, and the gradient of the logits

run() computes them as plain torch operations in 32 bits, or where `own` is true
through the C ABI's Python binding (train.cpp_amd/hip.py).
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 128  # elements that share a scale, along a row and in a weight down its rows too
TOP = 448.0  # the largest e4m3


def _hip():
    """This repository's binding; its folder's name has a dot, so it is loaded by its file."""
    if "traincpp_amd" not in sys.modules:
        pkg = Path(__file__).resolve().parent.parent / "train.cpp_amd"
        spec = importlib.util.spec_from_file_location("traincpp_amd", pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["traincpp_amd"] = mod
        spec.loader.exec_module(mod)
    from traincpp_amd import hip
    return hip


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one token through a layer of a small model, the smallest call: latency and launches
        {"name": "fp8_one_small", "op": "fp8", "type": "f32", "scales": "pow2", "K": 768, "M": 288, "N": 1},
        # a single request's decode step through the MLP's up projection of a 4096-wide model
        {"name": "fp8_decode_1", "op": "fp8", "type": "f32", "scales": "float", "K": 4096, "M": 14336, "N": 1},
        # a decode step of 16 requests through the attention's output projection
        {"name": "fp8_decode_16", "op": "fp8", "type": "bf16", "scales": "pow2", "K": 4096, "M": 4096, "N": 16},
        # a short prompt on a layer whose sizes fit no block
        {"name": "fp8_ragged", "op": "fp8", "type": "f16", "scales": "float", "K": 2050, "M": 1999, "N": 333},
        # long prompts, or a batch of training sequences; the weight as this framework quantizes it
        {"name": "fp8_4096_tokens", "op": "fp8", "type": "bf16", "scales": "pow2", "K": 4096, "M": 14336, "N": 4096},
        # the same size of batch on a weight whose scales a checkpoint brings
        {"name": "fp8_2048_tokens", "op": "fp8", "type": "f32", "scales": "float", "K": 4096, "M": 4096, "N": 2048},
        # the way back through the layer under adapters that are tuned, 512 tokens
        {"name": "fp8_back_512", "op": "fp8_back", "type": "f32", "scales": "pow2", "K": 4096, "M": 4096, "N": 512},
        # the same for a batch of sequences through the MLP's down projection, gradients in 16 bits
        {"name": "fp8_back_2048", "op": "fp8_back", "type": "bf16", "scales": "float", "K": 14336, "M": 4096, "N": 2048},
        # a few tokens on a small layer whose sizes fit no block
        {"name": "fp8_back_ragged", "op": "fp8_back", "type": "f32", "scales": "float", "K": 1000, "M": 777, "N": 61},
        # a short answer over a large vocabulary: few rows, each of them long
        {"name": "distill_short_wide", "op": "distill", "type": "f32", "V": 131071, "T": 61, "top": 20, "tau": 2.0,
         "alpha": 0.5},
        # a training batch with logits in 16 bits, the teacher's top 64
        {"name": "distill_8192", "op": "distill", "type": "bf16", "V": 32000, "T": 8192, "top": 64, "tau": 2.0,
         "alpha": 0.9},
        # the teacher's distribution alone, at its own temperature, over a vocabulary that fits no vector
        {"name": "distill_odd", "op": "distill", "type": "f16", "V": 5003, "T": 777, "top": 7, "tau": 1.0, "alpha": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: multiples of 128 or 8, or any number."""
    step = rng.choice([128, 128, 8, 1])
    return max(step, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["fp8", "fp8", "fp8_back", "distill"])
    if op == "distill":
        v = _width(rng, 500, 131072)
        return {"op": op, "type": rng.choice(list(DTYPES)), "V": v, "T": min(_log(rng, 8, 8192), (1 << 28) // v),
                "top": _log(rng, 1, 128), "tau": rng.choice([1.0, 2.0, 4.0, 1.5]), "alpha": rng.choice([1.0, 0.9, 0.5])}
    n = {"one": 1, "few": _log(rng, 2, 64), "many": _log(rng, 65, 4096)}[rng.choice(["one", "few", "many", "many"])]
    return {"op": op, "type": rng.choice(list(DTYPES)), "scales": rng.choice(["pow2", "float"]),
            "K": _width(rng, 64, 14336 if n <= 2048 else 4096), "M": _width(rng, 64, 14336), "N": n}


def _choices(case):
    """What of a case's inputs its sizes decide: a generator that starts the same for the same case."""
    return random.Random("/".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))


def _prompts(case):
    """Which rows are not counted: the first tokens of sequences of some 100."""
    rng, T, at, out = _choices(case), case["T"], 0, []
    while at < T:
        n = min(rng.randint(30, 170), T - at)
        out += [True] * (n // 4) + [False] * (n - n // 4)
        at += n
    return out


# ------------------------------------------------------------------ inputs

def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32) * std


def _ceil(a, b):
    return -(-a // b)


def _t(H, x):
    """The ggml descriptor of a torch tensor: ne[0] is torch's last dimension."""
    types = {torch.float32: H.TYPE_F32, torch.float16: H.TYPE_F16, torch.bfloat16: H.TYPE_BF16,
             torch.int32: H.TYPE_I32, torch.uint8: H.TYPE_I8}
    shape, stride = list(x.shape), list(x.stride())
    lead, es = 4 - x.dim(), x.element_size()
    span = max(n * s for n, s in zip(shape, stride))
    return H.tensor(x.data_ptr(), shape[::-1] + [1] * lead, [es * s for s in stride[::-1]] + [es * span] * lead,
                    types[x.dtype])


def _two(e):
    """2^e as a float, e from -126 to 127 (torch's own powers of two are a rounding off for some)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pow2_exponent(amax):
    """The exponent of the smallest power of two by which amax falls to 448 or less (-126 at least; 0 for a block of zeros)."""
    f, e = torch.frexp(amax)  # amax = f 2^e, f in [1/2, 1); 448 = 7/8 2^9
    e = (e - 9 + (f > 0.875).to(e.dtype)).clamp(min=-126)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _quantize(x):
    """Rows in blocks of 128: e4m3 values in 32 bits, and the exponents of their scales."""
    n, k = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(n, -1, BLOCK)
    e = _pow2_exponent(b.abs().amax(2))
    q = (b * _two(-e)[:, :, None]).to(torch.float8_e4m3fn)
    return q, e


def _values(q, e, k):
    """What the codes of _quantize stand for."""
    v = q.float() * _two(e)[:, :, None]
    return v.view(v.shape[0], -1)[:, :k]


def _weight(s):
    """The weight's values: codes [M, K] times their blocks' scales."""
    c = s["case"]
    scale = s["w_scale"]
    if c["scales"] == "pow2":  # a byte holds the exponent, 127 added
        scale = _two(scale.int() - 127)
    w = s["w"][:, :c["K"]].view(torch.float8_e4m3fn).float()
    scale = scale[:, :_ceil(c["K"], BLOCK)].repeat_interleave(BLOCK, 0)[:c["M"]]
    return w * scale.repeat_interleave(BLOCK, 1)[:, :c["K"]]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    c, op = case, case["op"]
    s = {"case": c, "op": op}
    H = _hip() if own else None
    if own:
        H.init(0)
    if op in ("fp8", "fp8_back"):
        K, M, N, dt = c["K"], c["M"], c["N"], DTYPES[c["type"]]
        kb, mb = _ceil(K, BLOCK), _ceil(M, BLOCK)
        # a layer's weights, rows of different size among them, in blocks of 128 x 128
        w = _normal(g, M, K, std=K ** -0.5) * torch.exp(_normal(g, M, 1, std=0.3))
        blocks = torch.nn.functional.pad(w, (0, -K % BLOCK, 0, -M % BLOCK)).view(mb, BLOCK, kb, BLOCK)
        amax = blocks.abs().amax((1, 3))
        if c["scales"] == "pow2":
            e = _pow2_exponent(amax)
            blocks = blocks * _two(-e)[:, None, :, None]
            s["w_scale"] = torch.full((mb, _ceil(kb, 4) * 4), 127, dtype=torch.uint8, device=DEVICE)
            s["w_scale"][:, :kb] = (e + 127).to(torch.uint8)
        else:
            s["w_scale"] = amax / TOP
            blocks = (blocks / s["w_scale"][:, None, :, None]).clamp(-TOP, TOP)
        codes = blocks.to(torch.float8_e4m3fn).view(torch.uint8).reshape(mb * BLOCK, kb * BLOCK)
        s["w"] = codes[:M].contiguous()  # rows of whole blocks, zeros past K
        del w, blocks, codes
        shape, out = ((N, K), (N, M)) if op == "fp8" else ((N, M), (N, K))
        # activations (or gradients) with a few channels far larger than the rest
        size = torch.exp(_normal(g, 1, shape[1], std=0.5))
        s["x"] = (_normal(g, *shape, std=1.0 if op == "fp8" else 1e-3) * size).to(dt)
        if own:
            xb = _ceil(shape[1], BLOCK)
            s["xq"] = torch.empty(N, xb * BLOCK, dtype=torch.uint8, device=DEVICE)
            s["x_scale"] = torch.empty(N, _ceil(xb, 4) * 4, dtype=torch.uint8, device=DEVICE)
            s["y"] = torch.empty(out, dtype=dt, device=DEVICE)
            s["t"] = {"w": H.fp8(_t(H, s["w"][:, :K]), _t(H, s["w_scale"][:, :kb])),
                      "xq": H.fp8(_t(H, s["xq"][:, :shape[1]]), _t(H, s["x_scale"][:, :xb])),
                      "x": _t(H, s["x"]), "y": _t(H, s["y"])}
        return s
    V, T, k, dt = c["V"], c["T"], c["top"], DTYPES[c["type"]]
    # the teacher's tokens of a row, all different, in falling order of their logits
    at = torch.randint(0, V, (T, 1), generator=g, device=DEVICE)
    step = torch.randint(1, max(V // k, 2), (T, 1), generator=g, device=DEVICE)
    ids = (at + step * torch.arange(k, device=DEVICE)) % V
    s["ids"] = ids.to(torch.int32)
    s["top"] = (_normal(g, T, k, std=2.0).sort(1, descending=True).values + 12.0).to(dt)
    # the student finds the same tokens likely, with errors
    logits = _normal(g, T, V, std=2.0)
    logits.scatter_add_(1, ids, (s["top"].float() - 3.0) * torch.rand(T, k, generator=g, device=DEVICE))
    s["logits"] = logits.to(dt)
    pick = torch.randint(0, k, (T,), generator=g, device=DEVICE)
    s["labels"] = s["ids"][torch.arange(T, device=DEVICE), pick].contiguous()
    s["labels"][torch.tensor(_prompts(c), device=DEVICE)] = -1
    s["dloss"] = torch.ones(1, device=DEVICE)
    if own:
        s["stats"], s["loss"] = torch.empty(T, 5, device=DEVICE), torch.empty(4, device=DEVICE)
        s["dlogits"] = torch.empty_like(s["logits"])
        s["t"] = {n: _t(H, s[n]) for n in ("logits", "labels", "ids", "top", "stats", "loss", "dloss", "dlogits")}
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    H, c, t = _hip(), s["case"], s["t"]
    if s["op"] == "distill":
        H.distill_loss(t["logits"], t["labels"], t["ids"], t["top"], c["tau"], c["alpha"], t["stats"], t["loss"])
        H.distill_loss_back(t["logits"], t["labels"], t["ids"], t["top"], t["stats"], t["loss"], t["dloss"], c["tau"],
                            c["alpha"], t["dlogits"])
        return {"loss": s["loss"], "dlogits": s["dlogits"]}
    if s["op"] == "fp8" and c["N"] <= H.FP8_MATVEC_MAX_N:
        H.fp8_matvec(t["w"], t["x"], t["y"])
        return {"y": s["y"]}
    H.fp8_quantize(t["x"], t["xq"])
    if s["op"] == "fp8":
        H.fp8_mul_mat(t["w"], t["xq"], t["y"])
        return {"y": s["y"]}
    H.fp8_mul_mat_back(t["w"], t["xq"], t["y"])
    return {"dx": s["y"]}


def _plain(s):
    c = s["case"]
    if s["op"] in ("fp8", "fp8_back"):
        x = _values(*_quantize(s["x"]), s["x"].shape[1])
        w = _weight(s)
        if s["op"] == "fp8":
            return {"y": (x @ w.t()).to(s["x"].dtype)}
        return {"dx": (x @ w).to(s["x"].dtype)}
    tau, alpha = c["tau"], c["alpha"]
    l, y, ids, z = s["logits"].float(), s["labels"].long(), s["ids"].long(), s["top"].float() / tau
    counted = y >= 0
    n = counted.sum()
    unit = counted.float()[:, None] / n
    zero = torch.zeros((), device=DEVICE)
    # the teacher's probabilities, and their logarithms
    z = z - z.amax(1, keepdim=True)
    logp = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    p = torch.exp(logp)
    m = l.amax(1, keepdim=True)
    l = l - m
    soft = l / tau
    e = torch.exp(soft)
    total = e.sum(1, keepdim=True)
    kl = (p * (logp - soft.gather(1, ids) + torch.log(total))).sum(1)
    kl = torch.where(counted, kl, zero).sum() / n
    d = (e / total) * unit * (alpha * tau)
    d.scatter_add_(1, ids, -p * unit * (alpha * tau))
    ce = zero
    if alpha < 1:
        e = torch.exp(l)
        total = e.sum(1, keepdim=True)
        at = y.clamp(min=0)[:, None]
        ce = (torch.log(total) - l.gather(1, at))[:, 0]
        ce = torch.where(counted, ce, zero).sum() / n
        d += (e / total) * unit * (1 - alpha)
        d.scatter_add_(1, at, -unit * (1 - alpha))
    loss = torch.stack([alpha * tau * tau * kl + (1 - alpha) * ce, kl, ce, n.float()])
    return {"loss": loss, "dlogits": (d * s["dloss"]).to(s["logits"].dtype)}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    e = 4 if c["type"] == "f32" else 2
    if c["op"] == "distill":
        counted = c["T"] - sum(_prompts(c))
        logits = c["V"] * (counted + c["T"])
        exps = (1 if c["alpha"] == 1.0 or c["tau"] == 1.0 else 2)
        return {"bytes": e * logits + (4 + e) * counted * c["top"] + 4 * c["T"], "flops": 8 * exps * counted * c["V"]}
    K, M, N = c["K"], c["M"], c["N"]
    scales = _ceil(K, BLOCK) * _ceil(M, BLOCK) * (1 if c["scales"] == "pow2" else 4)
    return {"bytes": K * M + scales + e * N * (K + M), "flops": 2 * K * M * N}


# ------------------------------------------------------------------ results in 64 bits

def _two64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3_round(v):
    """v of magnitude up to 448 to the nearest e4m3 (8 steps to a power of two, 2^-9 at least), ties to even."""
    _, e = torch.frexp(v)
    step = _two64((e - 4).clamp(min=-9))
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    c, D = case, torch.float64
    if c["op"] in ("fp8", "fp8_back"):
        K, M, N = c["K"], c["M"], c["N"]
        x = s["x"].to(D)
        for lo in range(0, x.shape[1], BLOCK):  # the quantizing is exact but for the codes' rounding
            part = x[:, lo:lo + BLOCK]
            top = part.abs().amax(1, keepdim=True)
            power = torch.ceil(torch.log2((top / TOP).clamp(min=2.0 ** -300))).long()
            power += (top > TOP * _two64(power)).long() - (top <= TOP * _two64(power - 1)).long()
            scale = torch.where(top > 0, _two64(power.clamp(min=-126)), torch.ones_like(top))
            x[:, lo:lo + BLOCK] = _e4m3_round(part / scale) * scale
        codes = s["w"].long()
        sign, expo, man = codes >> 7, (codes >> 3) & 15, (codes & 7).to(D)
        w = torch.where(expo > 0, (1 + man / 8) * _two64(expo - 7), man * 2.0 ** -9) * (1 - 2 * sign)
        scale = _two64(s["w_scale"].long() - 127) if c["scales"] == "pow2" else s["w_scale"].to(D)
        for i in range(_ceil(M, BLOCK)):
            for j in range(_ceil(K, BLOCK)):
                w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[i, j]
        w = w[:, :K]
        if c["op"] == "fp8":
            return {"y": torch.matmul(x, w.t().contiguous())}
        return {"dx": torch.matmul(x, w.contiguous())}
    T, tau, alpha = c["T"], c["tau"], c["alpha"]
    y, ids = s["labels"].long(), s["ids"].long()
    n = int((y >= 0).sum())
    d = torch.zeros(T, c["V"], dtype=D, device=DEVICE)
    kl = ce = 0.0
    for lo in range(0, T, 1024):
        use = (y[lo:lo + 1024] >= 0).nonzero()[:, 0] + lo
        l = s["logits"][use].to(D)
        rows = torch.arange(len(use), device=DEVICE)
        logp = torch.log_softmax(s["top"][use].to(D) / tau, 1)
        logq = torch.log_softmax(l / tau, 1)
        kl = kl + (torch.exp(logp) * (logp - logq.gather(1, ids[use]))).sum() / n
        part = torch.exp(logq)
        part.scatter_add_(1, ids[use], -torch.exp(logp))
        part *= alpha * tau / n
        if alpha < 1:
            logq = torch.log_softmax(l, 1)
            ce = ce - logq[rows, y[use]].sum() / n
            hard = torch.exp(logq)
            hard[rows, y[use]] -= 1
            part += hard * ((1 - alpha) / n)
        d[use] = part
    loss = [alpha * tau * tau * kl + (1 - alpha) * ce, kl, ce, n]
    return {"loss": torch.stack([torch.as_tensor(v, dtype=D, device=DEVICE) for v in loss]), "dlogits": d}
