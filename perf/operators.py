"""The operators of adapter tuning as cases to be timed and checked.

A case is a dict of plain values; its "op" says what a pass is:

  lora       low-rank adapters of the requests of one batch, added to the output
             of the projection they share: y = base + s B (A x)
  lora_back  their backward pass: dx = base + s A^T B^T dy and the gradients of
             every adapter's two matrices
  pref       the preference loss of pairs of sequences over logits, with the
             gradient of the logits
  adamw      one AdamW step over all tensors of a list, moments in 32 bits, or in
             8 bits (then the moments are read out as floats too, as a checkpoint
             does)

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
BLOCK = 256  # elements that share a scale in the 8-bit moments
ALIGN = 256  # elements: where the tensors of one buffer start


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
        {"name": "lora_one_small", "op": "lora", "type": "f32", "K": 768, "M": 288, "R": 8, "T": 1, "requests": 1,
         "adapters": 4},
        # a decode step: 64 requests of one token each on 16 adapters
        {"name": "lora_decode64", "op": "lora", "type": "f16", "K": 4096, "M": 4096, "R": 16, "T": 64, "requests": 64,
         "adapters": 16},
        # prompts and single tokens in one batch, the MLP's up projection, a wide rank
        {"name": "lora_mixed", "op": "lora", "type": "bf16", "K": 4096, "M": 14336, "R": 64, "T": 1001, "requests": 13,
         "adapters": 6},
        # a batch of training sequences, or long prompts, on one adapter
        {"name": "lora_4096_tokens", "op": "lora", "type": "f32", "K": 4096, "M": 4096, "R": 16, "T": 4096,
         "requests": 8, "adapters": 1},
        # the gradients of one adapted layer over 512 tokens
        {"name": "lora_back_512", "op": "lora_back", "type": "f32", "K": 4096, "M": 4096, "R": 16, "T": 512,
         "requests": 2, "adapters": 1},
        # three adapters tuned in one batch on a small layer whose sizes fit no tile
        {"name": "lora_back_ragged", "op": "lora_back", "type": "bf16", "K": 1000, "M": 777, "R": 20, "T": 1333,
         "requests": 7, "adapters": 3},
        # two pairs of short answers over a large vocabulary: few rows, each of them long
        {"name": "pref_short_wide", "op": "pref", "type": "f32", "V": 131071, "T": 61, "pairs": 2},
        # a batch of eight pairs with logits in 16 bits
        {"name": "pref_8_pairs", "op": "pref", "type": "bf16", "V": 32000, "T": 8192, "pairs": 8},
        # the tensors of 112 adapters of rank 16: many small ones, one step
        {"name": "adamw_adapters", "op": "adamw", "layout": "adapters", "n": 224, "K": 4096, "R": 16, "bits": 32,
         "grad": "f32"},
        # the weights, biases and norms of one 4096-wide layer, moments in 32 bits
        {"name": "adamw_layer", "op": "adamw", "layout": "layer", "n": 1, "K": 4096, "R": 14336, "bits": 32,
         "grad": "f32"},
        # the same layer with its moments in 8 bits and gradients in 16
        {"name": "adamw8_layer", "op": "adamw", "layout": "layer", "n": 1, "K": 4096, "R": 14336, "bits": 8,
         "grad": "bf16"},
        # tensors of every size, most of them odd
        {"name": "adamw8_odd", "op": "adamw", "layout": "odd", "n": 61, "K": 300000, "R": 1, "bits": 8, "grad": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: multiples of 128 or 8, or any number."""
    step = rng.choice([128, 128, 8, 1])
    return max(step, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["lora", "lora", "lora_back", "pref", "adamw"])
    if op == "lora":
        kind = rng.choice(["single", "mixed", "long"])
        c = {"op": op, "type": rng.choice(list(DTYPES)), "K": _width(rng, 64, 8192), "M": _width(rng, 64, 14336),
             "R": rng.choice([4, 8, 16, 16, 32, 64, _log(rng, 1, 128)])}
        if kind == "single":
            t = _log(rng, 1, 128)
            return {**c, "T": t, "requests": t, "adapters": _log(rng, 1, 32)}
        if kind == "mixed":
            q = _log(rng, 2, 32)
            return {**c, "T": q + _log(rng, 16, 2048), "requests": q, "adapters": _log(rng, 1, 16)}
        return {**c, "T": _log(rng, 256, 4096), "requests": rng.randint(1, 8), "adapters": rng.randint(1, 3)}
    if op == "lora_back":
        q = rng.randint(1, 8)
        return {"op": op, "type": rng.choice(list(DTYPES)), "K": _width(rng, 64, 8192), "M": _width(rng, 64, 8192),
                "R": rng.choice([4, 8, 16, 16, 32, 64, _log(rng, 1, 128)]), "T": q + _log(rng, 16, 4096),
                "requests": q, "adapters": rng.randint(1, 4)}
    if op == "pref":
        p, v = rng.randint(1, 8), _width(rng, 500, 131072)
        t = min(_log(rng, 8, 8192), (1 << 28) // v)
        return {"op": op, "type": rng.choice(list(DTYPES)), "V": v, "T": 2 * p + t, "pairs": p}
    layout = rng.choice(["adapters", "layer", "odd"])
    c = {"op": op, "layout": layout, "bits": rng.choice([8, 32]), "grad": rng.choice(list(DTYPES))}
    if layout == "adapters":
        return {**c, "n": 2 * _log(rng, 4, 224), "K": _width(rng, 256, 8192), "R": rng.choice([8, 16, 32, 64])}
    if layout == "layer":
        return {**c, "n": 1, "K": _width(rng, 256, 4096), "R": _width(rng, 256, 14336)}
    return {**c, "n": _log(rng, 1, 200), "K": _log(rng, 100, 1000000), "R": 1}


def _choices(case):
    """What of a case's inputs its sizes decide: a generator that starts the same for the same case."""
    return random.Random("/".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))


def _lengths(rng, total, parts):
    """`total` in `parts` whole numbers of 1 or more."""
    if parts == total:
        return [1] * parts
    cuts = sorted(rng.sample(range(1, total), parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _requests(case):
    """The requests' lengths and adapters. Every adapter that fits has a request; of
    three requests or more the last has none (the base model's own answer)."""
    rng = _choices(case)
    q, n = case["requests"], case["adapters"]
    lens = _lengths(rng, case["T"], q)
    ids = [i if i < n else rng.randrange(n) for i in range(q)]
    if q > 2:
        ids[-1] = -1
    return lens, ids


def _sequences(case):
    """The sequences' lengths and how many tokens of each, its prompt, are not counted."""
    lens = _lengths(_choices(case), case["T"], 2 * case["pairs"])
    return lens, [n // 4 for n in lens]


def _shapes(case):
    """The tensors' shapes, and which of them decay."""
    K, R = case["K"], case["R"]
    if case["layout"] == "adapters":
        return [((R, K) if i % 2 == 0 else (K, R), True) for i in range(case["n"])]
    if case["layout"] == "layer":
        return ([((K, K), True)] * 4 + [((R, K), True)] * 2 + [((K, R), True)] + [((K,), False)] * 3 + [((R,), False)])
    rng = _choices(case)
    return [((_log(rng, 1, K) + i % 2,), i % 3 != 0) for i in range(case["n"])]


# ------------------------------------------------------------------ inputs

def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32) * std


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _t(H, x):
    """The ggml descriptor of a torch tensor: ne[0] is torch's last dimension."""
    types = {torch.float32: H.TYPE_F32, torch.float16: H.TYPE_F16, torch.bfloat16: H.TYPE_BF16,
             torch.int32: H.TYPE_I32}
    shape, stride = list(x.shape), list(x.stride())
    lead, es = 4 - x.dim(), x.element_size()
    span = max(n * s for n, s in zip(shape, stride))
    return H.tensor(x.data_ptr(), shape[::-1] + [1] * lead, [es * s for s in stride[::-1]] + [es * span] * lead,
                    types[x.dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    c, op = case, case["op"]
    s = {"case": c, "op": op}
    H = _hip() if own else None
    if own:
        H.init(0)
    if op in ("lora", "lora_back"):
        K, M, R, T, n, dt = c["K"], c["M"], c["R"], c["T"], c["adapters"], DTYPES[c["type"]]
        lens, ids = _requests(c)
        s["start"], s["ids"] = _starts(lens), ids
        s["a"] = _normal(g, n, R, K, std=K ** -0.5).to(dt)
        s["b"] = _normal(g, n, M, R, std=0.05).to(dt)
        s["scale"] = torch.rand(n, generator=g, device=DEVICE) * 1.5 + 0.5
        s["x"] = _normal(g, T, K)
        s["start_d"], s["ids_d"] = _i32(s["start"]), _i32(ids)
        if own:
            s["set"] = H.lora_set(*(_t(H, s[k]) for k in ("a", "b", "scale", "start_d", "ids_d")))
            s["h"] = torch.empty(T, R, device=DEVICE)
        if op == "lora":
            s["base"] = _normal(g, T, M)
            if own:
                s["y"] = torch.empty(T, M, device=DEVICE)
                s["t"] = [_t(H, s[k]) for k in ("x", "base", "h", "y")]
            return s
        s["dy"] = _normal(g, T, M, std=1e-2)
        s["base"] = _normal(g, T, K, std=1e-2)
        s["h"] = torch.zeros(T, R, device=DEVICE)
        for q, a in enumerate(ids):  # what the forward pass left
            if a >= 0:
                rows = slice(s["start"][q], s["start"][q + 1])
                s["h"][rows] = s["x"][rows] @ s["a"][a].float().t()
        if own:
            s["g"], s["dx"] = torch.empty(T, R, device=DEVICE), torch.empty(T, K, device=DEVICE)
            s["da"], s["db"] = torch.empty(n, R, K, device=DEVICE), torch.empty(n, M, R, device=DEVICE)
            s["t"] = [_t(H, s[k]) for k in ("x", "h", "dy", "g", "base", "dx", "da", "db")]
    elif op == "pref":
        V, T, P, dt = c["V"], c["T"], c["pairs"], DTYPES[c["type"]]
        lens, prompt = _sequences(c)
        s["start"] = _starts(lens)
        s["logits"] = _normal(g, T, V, std=2.0).to(dt)
        s["labels"] = torch.randint(0, V, (T,), generator=g, device=DEVICE, dtype=torch.int32)
        # the model finds its own answers likelier than chance
        s["logits"][torch.arange(T, device=DEVICE), s["labels"].long()] += 12.0
        skip = torch.cat([torch.arange(n, device=DEVICE) < p for n, p in zip(lens, prompt)])
        s["labels"][skip] = -1
        s["seq"] = torch.repeat_interleave(torch.arange(2 * P, device=DEVICE), torch.tensor(lens, device=DEVICE))
        counted = torch.tensor([n - p for n, p in zip(lens, prompt)], device=DEVICE)
        # the reference model's sums lie near the model's own
        s["ref"] = _reference_sums(s) + _normal(g, 2 * P) * counted.float().sqrt() * 0.5
        s["start_d"] = _i32(s["start"])
        s["dloss"] = torch.ones(1, device=DEVICE)
        if own:
            s["dlogits"] = torch.empty_like(s["logits"])
            for k, n in (("lse", T), ("logp", 2 * P), ("slope", P), ("loss", 1)):
                s[k] = torch.empty(n, device=DEVICE)
            s["t"] = {k: _t(H, s[k]) for k in ("logits", "labels", "start_d", "ref", "lse", "logp", "slope", "loss",
                                               "dloss", "dlogits")}
    else:
        shapes = _shapes(c)
        n = [math.prod(shape) for shape, _ in shapes]
        s["n"], s["decay"] = n, [1.0 if decay else 0.0 for _, decay in shapes]
        at = s["at"] = [0]
        for k in n:
            at.append(at[-1] + -(-k // ALIGN) * ALIGN)
        s["p"], s["grad"] = _normal(g, at[-1], std=0.02), _normal(g, at[-1], std=1e-3).to(DTYPES[c["grad"]])
        s["hyper"] = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1, "step": 1000}
        # moments after many steps of gradients like these
        s["m"] = _normal(g, at[-1], std=2e-4)
        s["v"] = (_normal(g, at[-1]) ** 2 * 0.9 + 0.1) * 1e-6
        if c["bits"] == 8:
            s["m_scale"], s["v_scale"] = (torch.zeros(at[-1] // BLOCK, device=DEVICE) for _ in range(2))
            floats = {"m": s["m"], "v": torch.sqrt(s["v"])}
            s["m"], s["v"] = (torch.zeros(at[-1], device=DEVICE, dtype=dt) for dt in (torch.int8, torch.uint8))
            for i in range(len(n)):
                for k, pack in (("m", _pack_m), ("v", _pack_v)):
                    _store(s, k, i, *pack(_piece(s, floats[k], i)))
            if own:
                s["m_out"], s["v_out"] = (torch.zeros(at[-1], device=DEVICE) for _ in range(2))
        if own:
            grad_type = {"f32": H.TYPE_F32, "f16": H.TYPE_F16, "bf16": H.TYPE_BF16}[c["grad"]]

            def ptr(k, i):
                return s[k].data_ptr() + (at[i] // BLOCK if "scale" in k else at[i]) * s[k].element_size()

            states = ("m", "v") if c["bits"] == 32 else ("m", "v", "m_scale", "v_scale", "m_out", "v_out")
            s["plan"] = H.AdamW([dict(n=n[i], decay=s["decay"][i], grad_type=grad_type, param=ptr("p", i),
                                      **{k: ptr(k, i) for k in ("grad",) + states}) for i in range(len(n))], c["bits"])
    return s


def _reference_sums(s):
    """Each sequence's log-probability, a few rows at a time."""
    T = s["case"]["T"]
    lps = torch.empty(T, device=DEVICE)
    for i in range(0, T, 512):
        l, y = s["logits"][i:i + 512].float(), s["labels"][i:i + 512].long()
        lp = l.gather(1, y.clamp(min=0)[:, None])[:, 0] - torch.log(torch.exp(l - 20.0).sum(1)) - 20.0
        lps[i:i + 512] = torch.where(y >= 0, lp, torch.zeros_like(lp))
    return torch.stack([lps[lo:hi].sum() for lo, hi in zip(s["start"], s["start"][1:])])


def _piece(s, x, i):
    """Tensor i of an arena."""
    return x[s["at"][i]:s["at"][i] + s["n"][i]]


def _scales(s, k, i):
    lo = s["at"][i] // BLOCK
    return s[k + "_scale"][lo:lo - (-s["n"][i] // BLOCK)]


def _store(s, k, i, code, scale):
    _piece(s, s[k], i).copy_(code)
    _scales(s, k, i).copy_(scale)


# ------------------------------------------------------------------ the 8-bit moments
#
# Blocks of 256 elements share a scale, the largest magnitude of the block:
#   first moment   m       = scale * sign(c) * (c / 127)^2
#   second moment  sqrt(v) = scale * (c / 255)^2, with c at least 1 where v > 0

def _blocks(x):
    pad = -x.numel() % BLOCK
    x = x.reshape(-1)
    return (torch.cat([x, x.new_zeros(pad)]) if pad else x).view(-1, BLOCK)


def _inverse(scale):
    tiny = 2.0 ** -126
    return torch.where(scale >= tiny, 1.0 / torch.where(scale >= tiny, scale, torch.ones_like(scale)),
                       torch.zeros_like(scale))


def _pack_m(m):
    b = _blocks(m)
    scale = b.abs().amax(1)
    inv = _inverse(scale)
    c = torch.round(torch.sqrt(b.abs() * inv[:, None]) * 127.0)
    c = torch.where(b < 0, -c, c).to(torch.int8)
    return c.reshape(-1)[:m.numel()].clone(), torch.where(inv > 0, scale, torch.zeros_like(scale))


def _pack_v(u):
    b = _blocks(u)
    scale = b.amax(1)
    inv = _inverse(scale)
    r = b * inv[:, None]
    c = torch.round(torch.sqrt(r) * 255.0)
    c = torch.where(r > 0, c.clamp(min=1.0), c).to(torch.uint8)
    return c.reshape(-1)[:u.numel()].clone(), torch.where(inv > 0, scale, torch.zeros_like(scale))


def _unpack_m(code, scale, dtype=torch.float32):
    c = _blocks(code.to(dtype))
    m = c.abs() * c * scale.to(dtype)[:, None]
    return (m * _f32_constant(1.0 / 127 ** 2, dtype)).reshape(-1)[:code.numel()]


def _unpack_u(code, scale, dtype=torch.float32):
    c = _blocks(code.to(dtype))
    u = c * c * scale.to(dtype)[:, None]
    return (u * _f32_constant(1.0 / 255 ** 2, dtype)).reshape(-1)[:code.numel()]


def _f32_constant(x, dtype):
    return x if dtype == torch.float64 else float(torch.tensor(x, dtype=torch.float32))


# ------------------------------------------------------------------ one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    H, op = _hip(), s["op"]
    if op == "lora":
        H.lora(s["set"], *s["t"])
        return {"y": s["y"], "h": s["h"]}
    if op == "lora_back":
        H.lora_back(s["set"], *s["t"])
        return {"dx": s["dx"], "da": s["da"], "db": s["db"]}
    if op == "pref":
        t = s["t"]
        H.preference_loss(t["logits"], t["labels"], t["start_d"], t["ref"], 0.1, 0.05, t["lse"], t["logp"],
                          t["slope"], t["loss"])
        H.preference_loss_back(t["logits"], t["labels"], t["start_d"], t["lse"], t["slope"], t["dloss"], 0.1,
                               t["dlogits"])
        return {"loss": s["loss"], "logp": s["logp"], "dlogits": s["dlogits"]}
    s["plan"].step(**s["hyper"])
    if s["case"]["bits"] == 32:
        return {"p": s["p"], "m": s["m"], "v": s["v"]}
    s["plan"].moments()
    return {"p": s["p"], "m": s["m_out"], "v": s["v_out"]}


def _plain(s):
    op, c = s["op"], s["case"]
    if op in ("lora", "lora_back"):
        a, b = s["a"].float(), s["b"].float()
        spans = [(i, s["start"][q], s["start"][q + 1]) for q, i in enumerate(s["ids"]) if i >= 0]
    if op == "lora":
        if c["T"] == c["requests"]:  # one token each: all requests at once
            ids = s["ids_d"].long()
            with_one = ids >= 0
            ids = ids.clamp(min=0)
            h = (a[ids] * s["x"][:, None, :]).sum(2) * with_one[:, None]
            return {"y": s["base"] + (b[ids] * h[:, None, :]).sum(2) * s["scale"][ids][:, None], "h": h}
        y, h = s["base"].clone(), torch.zeros(c["T"], c["R"], device=DEVICE)
        for i, lo, hi in spans:
            h[lo:hi] = s["x"][lo:hi] @ a[i].t()
            y[lo:hi] += (h[lo:hi] @ b[i].t()) * s["scale"][i]
        return {"y": y, "h": h}
    if op == "lora_back":
        dx, da, db = s["base"].clone(), torch.zeros(a.shape, device=DEVICE), torch.zeros(b.shape, device=DEVICE)
        for i, lo, hi in spans:
            g = (s["dy"][lo:hi] @ b[i]) * s["scale"][i]
            dx[lo:hi] += g @ a[i]
            da[i] += g.t() @ s["x"][lo:hi]
            db[i] += (s["dy"][lo:hi].t() @ s["h"][lo:hi]) * s["scale"][i]
        return {"dx": dx, "da": da, "db": db}
    if op == "pref":
        P, beta, e = c["pairs"], 0.1, 0.05
        l, y = s["logits"].float(), s["labels"].long()
        counted, at = y >= 0, y.clamp(min=0)[:, None]
        top = l.amax(1, keepdim=True)
        lse = top + torch.log(torch.exp(l - top).sum(1, keepdim=True))
        lp = torch.where(counted, (l.gather(1, at) - lse)[:, 0], torch.zeros((), device=DEVICE))
        logp = torch.stack([lp[lo:hi].sum() for lo, hi in zip(s["start"], s["start"][1:])])
        ratio = (logp - s["ref"]).view(P, 2)
        z = beta * (ratio[:, 0] - ratio[:, 1])
        up, down = _softplus(-z), _softplus(z)
        loss = ((1 - e) * up + e * down).mean().reshape(1)
        slope = e * torch.sigmoid(z) - (1 - e) * torch.sigmoid(-z)
        w = torch.stack([slope, -slope], 1).reshape(-1) * (beta / P) * s["dloss"]
        w = torch.where(counted, w[s["seq"]], torch.zeros((), device=DEVICE))[:, None]
        dl = torch.exp(l - lse) * -w
        dl.scatter_add_(1, at, w)
        return {"loss": loss, "logp": logp, "dlogits": dl.to(s["logits"].dtype)}
    h = s["hyper"]
    b1, b2 = h["beta1"], h["beta2"]
    if c["bits"] == 8:
        out = {"p": s["p"], "m": torch.zeros_like(s["p"]), "v": torch.zeros_like(s["p"])}
    for i, n in enumerate(s["n"]):
        p, grad = _piece(s, s["p"], i), _piece(s, s["grad"], i).float()
        m, v = _piece(s, s["m"], i), _piece(s, s["v"], i)
        if c["bits"] == 8:
            m, u = _unpack_m(m, _scales(s, "m", i)), _unpack_u(v, _scales(s, "v", i))
            v = u * u
        m = m * b1 + grad * (1 - b1)
        v = v * b2 + (grad * grad) * (1 - b2)
        u = torch.sqrt(v)
        p.mul_(1 - h["lr"] * h["weight_decay"] * s["decay"][i])
        p.sub_((m / (u * (1 - b2 ** h["step"]) ** -0.5 + h["eps"])) * (h["lr"] / (1 - b1 ** h["step"])))
        if c["bits"] == 32:
            _piece(s, s["m"], i).copy_(m)
            _piece(s, s["v"], i).copy_(v)
            continue
        _store(s, "m", i, *_pack_m(m))
        _store(s, "v", i, *_pack_v(u))
        _piece(s, out["m"], i).copy_(_unpack_m(_piece(s, s["m"], i), _scales(s, "m", i)))
        u = _unpack_u(_piece(s, s["v"], i), _scales(s, "v", i))
        _piece(s, out["v"], i).copy_(u * u)
    return {"p": s["p"], "m": s["m"], "v": s["v"]} if c["bits"] == 32 else out


def _softplus(z):
    return z.clamp(min=0) + torch.log1p(torch.exp(-z.abs()))


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, op = case, case["op"]
    if op in ("lora", "lora_back"):
        K, M, R, T = c["K"], c["M"], c["R"], c["T"]
        e = 4 if c["type"] == "f32" else 2
        lens, ids = _requests(c)
        used = len({i for i in ids if i >= 0})
        tokens = sum(n for n, i in zip(lens, ids) if i >= 0)  # the others only pass through
        if op == "lora":
            return {"bytes": 4 * (tokens * K + 2 * T * M + T * R) + e * used * R * (K + M) + 4 * used,
                    "flops": 2 * tokens * R * (K + M)}
        # dy, x, h and the adapters read, dx's base read and dx written, both gradients written
        grads = 4 * c["adapters"] * R * (K + M)
        return {"bytes": 4 * (tokens * (M + K + R) + 2 * T * K) + e * used * R * (K + M) + grads,
                "flops": 4 * tokens * R * (K + M)}
    if op == "pref":
        e = 4 if c["type"] == "f32" else 2
        lens, prompt = _sequences(c)
        counted = sum(lens) - sum(prompt)
        return {"bytes": e * c["V"] * (counted + c["T"]) + 4 * c["T"], "flops": 8 * counted * c["V"]}
    n = sum(math.prod(shape) for shape, _ in _shapes(c))
    e = 4 if c["grad"] == "f32" else 2
    if c["bits"] == 32:
        return {"bytes": n * (8 + e + 16), "flops": 14 * n}
    return {"bytes": n * (8 + e + 4 + 8) + n // BLOCK * 16, "flops": 30 * n}


# ------------------------------------------------------------------ results in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op, c, D = s["op"], case, torch.float64
    if op in ("lora", "lora_back"):
        T, n, R = c["T"], c["adapters"], c["R"]
        x, a, b, sc = (s[k].to(D) for k in ("x", "a", "b", "scale"))
        base = s["base"].to(D)
        h = torch.zeros(T, R, dtype=D, device=DEVICE)
        first, da, db = base.clone(), torch.zeros_like(a), torch.zeros_like(b)
        for q, i in enumerate(s["ids"]):
            rows = slice(s["start"][q], s["start"][q + 1])
            if i < 0:
                continue
            if op == "lora":
                h[rows] = torch.matmul(x[rows], a[i].t().contiguous())
                first[rows] = base[rows] + sc[i] * torch.matmul(h[rows], b[i].t().contiguous())
                continue
            dy, hq = s["dy"][rows].to(D), s["h"][rows].to(D)
            first[rows] = base[rows] + torch.matmul(torch.matmul(dy, b[i]) * sc[i], a[i])
            da[i] += torch.matmul((torch.matmul(dy, b[i]) * sc[i]).t().contiguous(), x[rows])
            db[i] += torch.matmul(dy.t().contiguous(), hq) * sc[i]
        return {"y": first, "h": h} if op == "lora" else {"dx": first, "da": da, "db": db}
    if op == "pref":
        P, T = c["pairs"], c["T"]
        y = s["labels"].long()
        rows = []
        logp = torch.zeros(2 * P, dtype=D, device=DEVICE)
        for lo, hi, q in zip(s["start"], s["start"][1:], range(2 * P)):
            l = torch.log_softmax(s["logits"][lo:hi].to(D), 1)
            use = (y[lo:hi] >= 0).nonzero()[:, 0]
            logp[q] = l[use, y[lo:hi][use]].sum()
        gap = logp - s["ref"].to(D)
        loss, weight = 0.0, []
        for i in range(P):
            z = 0.1 * (gap[2 * i] - gap[2 * i + 1])
            loss = loss + (0.95 * torch.log1p(torch.exp(-z)) + 0.05 * torch.log1p(torch.exp(z))) / P
            k = 0.1 / P * (0.05 - 1 / (1 + torch.exp(z)))
            weight += [k, -k]
        for lo, hi, q in zip(s["start"], s["start"][1:], range(2 * P)):
            d = -torch.softmax(s["logits"][lo:hi].to(D), 1)
            use = y[lo:hi] >= 0
            d[use.nonzero()[:, 0], y[lo:hi][use]] += 1
            rows.append(d * (weight[q] * use.to(D))[:, None])
        return {"loss": loss.reshape(1), "logp": logp, "dlogits": torch.cat(rows)}
    h = s["hyper"]
    p, m, v = (s[k].to(D) for k in ("p", "m", "v"))  # the gaps between tensors stay as they are
    for i in range(len(s["n"])):
        grad, q = _piece(s, s["grad"], i).to(D), _piece(s, p, i)
        if c["bits"] == 32:
            mi, vi = _piece(s, m, i), _piece(s, v, i)
        else:
            mi = _unpack_m(_piece(s, s["m"], i), _scales(s, "m", i), D)
            vi = _unpack_u(_piece(s, s["v"], i), _scales(s, "v", i), D) ** 2
        mi = h["beta1"] * mi + (1 - h["beta1"]) * grad
        vi = h["beta2"] * vi + (1 - h["beta2"]) * grad ** 2
        mh, vh = mi / (1 - h["beta1"] ** h["step"]), vi / (1 - h["beta2"] ** h["step"])
        step = h["lr"] * mh / (torch.sqrt(vh) + h["eps"])
        q.copy_(q - h["lr"] * h["weight_decay"] * s["decay"][i] * q - step)
        _piece(s, m, i).copy_(mi)
        _piece(s, v, i).copy_(vi)
    # the 8-bit moments are whole codes: next to a boundary between two of them 64 bits say nothing
    return {"p": p, "m": m if c["bits"] == 32 else None, "v": v if c["bits"] == 32 else None}
