"""The operators between mhc_pre_clamp_sinkhorn and mhc_post: the layer norm
of the sublayer's input, the gated feed-forward block and the dropout of its
output, as programs that train or serve an mHC model run them.

A case is one pass: a forward call (``train`` false: serving) or a forward
and its backward (``train`` true), inputs resident on the GPU.  With ``own``
false, ``run`` computes the formulas with elementary torch operations in 32
bits; with ``own`` true it calls ``FlagOS_mhc.sublayer``.  ``exact`` is the
same in 64 bits, written apart.

Keys of a case:
  op      "norm", "ffn" or "dropout"
  T, D    tokens and width; F (op "ffn"): hidden width
  dtype   of the activations (and of the feed-forward weights)
  wdtype  (op "norm") of the norm's weight and bias
  act     (op "ffn") the gate's activation
  p       (op "dropout") probability of dropping
  train   forward and backward instead of the forward alone
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-5
_DEV = "cuda"


def _norm(name, T, D, dtype="bf16", wdtype="f32", train=True):
    return _named(name, dict(op="norm", T=T, D=D, dtype=dtype, wdtype=wdtype, train=train))


def _ffn(name, T, D, F, dtype="bf16", act="silu", train=True):
    return _named(name, dict(op="ffn", T=T, D=D, F=F, dtype=dtype, act=act, train=train))


def _drop(name, T, D, dtype="bf16", p=0.1, train=True):
    return _named(name, dict(op="dropout", T=T, D=D, dtype=dtype, p=p, train=train))


def _named(name, c):
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of a decoding loop: the norm before a sublayer
        _norm("norm_decode", 1, 7168, train=False),
        # a small fp32 model's training step
        _norm("norm_train_f32", 1024, 256, "f32"),
        # fp16 training, ragged tokens, rows that are no multiple of 16 bytes wide
        _norm("norm_train_odd_f16", 2049, 1003, "f16", "f16"),
        # the benchmark's batch: 65536 tokens at width 7168, forward and backward
        _norm("norm_train_large", 65536, 7168),
        # one token of a decoding loop: the weights are read once for a single row
        _ffn("ffn_decode_t1", 1, 7168, 18432, train=False),
        # a decoding batch of 64 sequences
        _ffn("ffn_decode_t64", 64, 4096, 11008, train=False),
        # a short prompt of odd length in fp16, rows that are no multiple of 16 bytes wide
        _ffn("ffn_prefill_odd_f16", 777, 1003, 2677, "f16", "gelu", train=False),
        # a small model's training step in fp32
        _ffn("ffn_train_f32", 1021, 512, 1408, "f32", "gelu_tanh"),
        # a middle-sized model's training step, ragged tokens
        _ffn("ffn_train", 4099, 2048, 5632),
        # a large model's training step
        _ffn("ffn_train_large", 16384, 7168, 18432),
        # a small fp32 model's training step
        _drop("dropout_train_f32", 1021, 255, "f32", 0.5),
        # the benchmark's batch, forward and backward
        _drop("dropout_train_large", 65536, 7168),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: usually a multiple of 64, now and then any number."""
    d = _log_int(rng, lo, hi)
    return d if d < 64 or rng.random() < 0.3 else d // 64 * 64


def draw(rng):
    op = rng.choice(["norm", "norm", "ffn", "ffn", "ffn", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    # fp32 rows hold twice the bytes: half the tokens at most
    top = 65536 if dtype != "f32" else 32768
    if op == "norm":
        return _norm(None, _log_int(rng, 1, top), _width(rng, 128, 7168), dtype,
                     rng.choice([dtype, "f32"]), rng.random() < 0.7)
    if op == "dropout":
        return _drop(None, _log_int(rng, 64, top), _width(rng, 128, 7168), dtype,
                     round(rng.uniform(0.02, 0.6), 3), rng.random() < 0.7)
    D = _width(rng, 128, 7168)
    F = max(128, int(D * rng.uniform(2.0, 3.5)))
    F = F if rng.random() < 0.3 else (F + 63) // 64 * 64
    F = min(F, 18432)
    train = rng.random() < 0.6
    T = _log_int(rng, 16 if train else 1, 16384 if dtype != "f32" else 2048)
    return _ffn(None, T, D, F, dtype, rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]), train)


# ---- inputs -------------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]
    T, D = case["T"], case["D"]

    def randn(*shape, scale=1.0, to=dt):
        return (torch.randn(*shape, device=_DEV, generator=g) * scale).to(to)

    s = {}
    if case["op"] == "norm":
        # what mhc_pre hands on: columns of different sizes, a few of them large, and an offset
        col = torch.exp(0.5 * torch.randn(D, device=_DEV, generator=g))
        col[:: max(1, D // 4)] *= 8.0
        off = 0.3 * torch.randn(D, device=_DEV, generator=g)
        x = torch.randn(T, D, device=_DEV, generator=g)
        s["x"] = x.mul_(col).add_(off).to(dt)
        wd = _DT[case["wdtype"]]
        s["weight"] = (1.0 + 0.2 * torch.randn(D, device=_DEV, generator=g)).to(wd)
        s["bias"] = (0.1 * torch.randn(D, device=_DEV, generator=g)).to(wd)
        if case["train"]:
            s["grad"] = randn(T, D)
    elif case["op"] == "ffn":
        F = case["F"]
        s["x"] = randn(T, D)
        s["w_gate"] = randn(F, D, scale=D ** -0.5)
        s["w_up"] = randn(F, D, scale=D ** -0.5)
        s["w_down"] = randn(D, F, scale=F ** -0.5)
        if case["train"]:
            s["grad"] = randn(T, D)
    else:
        s["x"] = randn(T, D)
        if case["train"]:
            s["grad"] = randn(T, D)
        # the number generator's key and position come from the program's own bookkeeping
        s["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) & 0x7FFFFFFFFFFFFFFF
        s["offset"] = seed % 1000 + 1
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    return s


# ---- the plain form ---------------------------------------------------------------

def _plain_norm(s):
    c = s["case"]
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = (xc.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    xhat = xc * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not c["train"]:
        return [y]
    gy = s["grad"].float()
    gw = (gy * xhat).sum(0)
    gb = gy.sum(0)
    g = gy * w
    gx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return [y, gx.to(s["x"].dtype), gw, gb]


_SQRT_HALF = math.sqrt(0.5)
_INV_SQRT_2PI = 1.0 / math.sqrt(2.0 * math.pi)
_GT0, _GT1 = math.sqrt(2.0 / math.pi), 0.044715


def _plain_act(kind, g):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * _SQRT_HALF))
    if kind == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(_GT0 * (g + _GT1 * g * g * g)))
    return torch.clamp(g, min=0.0)


def _plain_act_grad(kind, g):
    if kind == "silu":
        sg = torch.sigmoid(g)
        return sg * (1.0 + g * (1.0 - sg))
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(g * _SQRT_HALF)) + g * _INV_SQRT_2PI * torch.exp(-0.5 * g * g)
    if kind == "gelu_tanh":
        t = torch.tanh(_GT0 * (g + _GT1 * g * g * g))
        return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * _GT0 * (1.0 + 3.0 * _GT1 * g * g)
    return (g > 0).to(g.dtype)


def _plain_ffn(s):
    c = s["case"]
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g = x @ wg.t()
    u = x @ wu.t()
    a = _plain_act(c["act"], g)
    h = a * u
    out = (h @ wd.t()).to(dt)
    if not c["train"]:
        return [out]
    go = s["grad"].float()
    gh = go @ wd
    gwd = go.t() @ h
    gu = gh * a
    gg = gh * u * _plain_act_grad(c["act"], g)
    gx = gg @ wg + gu @ wu
    return [out, gx.to(dt), (gg.t() @ x).to(dt), (gu.t() @ x).to(dt), gwd.to(dt)]


_M32 = 0xFFFFFFFF


def _plain_philox(n_groups, seed, offset, device):
    """Philox4x32-10 (Salmon et al., SC 2011) in 64-bit integers: the four
    words of each group, key = seed, counter = (group, offset)."""
    i = torch.arange(n_groups, dtype=torch.int64, device=device)
    c0, c1 = i & _M32, i >> 32
    c2 = torch.full_like(i, offset & _M32)
    c3 = torch.full_like(i, (offset >> 32) & _M32)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(10):
        # products of two 32-bit numbers wrap modulo 2^64, which keeps every bit
        p0 = c0 * 0xD2511F53
        p1 = c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0 = (k0 + 0x9E3779B9) & _M32
        k1 = (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), -1)


def _threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def _plain_dropout(s):
    c = s["case"]
    x = s["x"]
    n = x.numel()
    words = _plain_philox((n + 7) // 8, s["seed"], s["offset"], x.device)
    halves = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:n]
    thr = _threshold(c["p"])
    keep = (halves >= thr).reshape(x.shape)
    scale = 65536.0 / (65536 - thr)
    out = [torch.where(keep, x.float() * scale, 0.0).to(x.dtype)]
    if c["train"]:
        out.append(torch.where(keep, s["grad"].float() * scale, 0.0).to(x.dtype))
    return out


# ---- the framework's operators -------------------------------------------------------

def _sublayer():
    import importlib
    import os
    import sys

    if "FlagOS_mhc.sublayer" not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flagos-mhc_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        importlib.import_module("FlagOS_mhc.sublayer")
    return sys.modules["FlagOS_mhc.sublayer"]


def _own_norm(s):
    c, lib = s["case"], _sublayer()
    if not c["train"]:
        return [lib.layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS)["y"]]
    f = lib.layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS, need_backward=True)
    gx, gw, gb = lib.layer_norm_backward(s["grad"], s["x"], s["weight"], f["mean"], f["rstd"])
    return [f["y"], gx, gw, gb]


def _own_ffn(s):
    c, lib = s["case"], _sublayer()
    args = (s["x"], s["w_gate"], s["w_up"], s["w_down"])
    if not c["train"]:
        return [lib.gated_ffn(*args, activation=c["act"])["out"]]
    f = lib.gated_ffn(*args, activation=c["act"], need_backward=True)
    g = lib.gated_ffn_backward(s["grad"], *args, f["gate"], f["up"], f["hidden"], activation=c["act"])
    return [f["out"], *g]


def _own_dropout(s):
    c, lib = s["case"], _sublayer()
    out = [lib.dropout(s["x"], c["p"], s["seed"], s["offset"])]
    if c["train"]:
        out.append(lib.dropout_backward(s["grad"], c["p"], s["seed"], s["offset"]))
    return out


_PLAIN = {"norm": _plain_norm, "ffn": _plain_ffn, "dropout": _plain_dropout}
_OWN = {"norm": _own_norm, "ffn": _own_ffn, "dropout": _own_dropout}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


# ---- floors ------------------------------------------------------------------------

def work(case):
    T, D, e = case["T"], case["D"], _SIZE[case["dtype"]]
    if case["op"] == "norm":
        w = D * _SIZE[case["wdtype"]]
        if not case["train"]:
            return {"bytes": 2 * T * D * e + 2 * w, "flops": 8 * T * D}
        # x and the gradient read, y and x's gradient written; weight, bias and their fp32 gradients
        return {"bytes": 4 * T * D * e + 2 * w + 8 * D, "flops": 22 * T * D}
    if case["op"] == "ffn":
        F = case["F"]
        fwd = 6 * T * D * F
        if not case["train"]:
            return {"bytes": (2 * T * D + 3 * D * F) * e, "flops": fwd}
        return {"bytes": (4 * T * D + 6 * D * F) * e, "flops": 3 * fwd}
    n = (4 if case["train"] else 2) * T * D
    return {"bytes": n * e, "flops": n // 2}


# ---- the definition in 64 bits -----------------------------------------------------------

def _exact_norm(s, case):
    T, D = s["x"].shape
    w, b = s["weight"].double(), s["bias"].double()
    y = torch.empty(T, D, dtype=torch.float64, device=_DEV)
    gx = torch.empty_like(y) if case["train"] else None
    gw = torch.zeros(D, dtype=torch.float64, device=_DEV)
    gb = torch.zeros(D, dtype=torch.float64, device=_DEV)
    for lo in range(0, T, 8192):
        rows = slice(lo, min(lo + 8192, T))
        x = s["x"][rows].double()
        mu = x.sum(1, keepdim=True) / D
        sd = torch.sqrt(((x - mu) ** 2).sum(1, keepdim=True) / D + _EPS)
        n = (x - mu) / sd
        y[rows] = n * w + b
        if case["train"]:
            d = s["grad"][rows].double()
            gw += (d * n).sum(0)
            gb += d.sum(0)
            q = d * w
            gx[rows] = (q - q.sum(1, keepdim=True) / D - n * ((q * n).sum(1, keepdim=True) / D)) / sd
    return [y, gx, gw, gb] if case["train"] else [y]


def _exact_act(kind, z):
    """(act(z), act'(z)) in 64 bits."""
    if kind == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return z * e, e + z * e * (1.0 - e)
    if kind == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        # 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v))
        v = k * (z + 0.044715 * z ** 3)
        e = 1.0 / (1.0 + torch.exp(-2.0 * v))
        return z * e, e + z * 2.0 * e * (1.0 - e) * k * (1.0 + 3 * 0.044715 * z ** 2)
    pos = z > 0
    return torch.where(pos, z, 0.0), pos.double()


def _exact_ffn(s, case):
    x, wg, wu, wd = (s[k].double() for k in ("x", "w_gate", "w_up", "w_down"))
    z = torch.mm(x, wg.t().contiguous())
    u = torch.mm(x, wu.t().contiguous())
    a, da = _exact_act(case["act"], z)
    h = a * u
    out = torch.mm(h, wd.t().contiguous())
    if not case["train"]:
        return [out]
    d = s["grad"].double()
    dh = torch.mm(d, wd)
    dz = dh * u * da
    du = dh * a
    del a, da, z, u, dh
    return [out, torch.mm(dz, wg) + torch.mm(du, wu), torch.mm(dz.t().contiguous(), x),
            torch.mm(du.t().contiguous(), x), torch.mm(d.t().contiguous(), h)]


def _mul_hi_lo(a, m):
    """High and low 32 bits of a * m (a a tensor, m a number, both below 2^32), by 16-bit halves."""
    ah, al, mh, ml = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
    low = al * ml
    mid = ah * ml + (low >> 16)
    mid2 = al * mh + (mid & 0xFFFF)
    return ah * mh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_dropout(s, case):
    n = s["x"].numel()
    thr = _threshold(case["p"])
    seed, off = s["seed"], s["offset"]
    names = ["x", "grad"] if case["train"] else ["x"]
    outs = [torch.zeros(n, dtype=torch.float64, device=_DEV) for _ in names]
    step = 1 << 26
    for lo in range(0, n, step):
        hi = min(lo + step, n)
        grp = torch.arange(lo // 8, (hi + 7) // 8, device=_DEV, dtype=torch.int64)
        ctr = [grp % (1 << 32), grp // (1 << 32), torch.full_like(grp, off % (1 << 32)),
               torch.full_like(grp, off // (1 << 32))]
        key = [seed % (1 << 32), seed // (1 << 32)]
        for r in range(10):
            h0, l0 = _mul_hi_lo(ctr[0], 0xD2511F53)
            h1, l1 = _mul_hi_lo(ctr[2], 0xCD9E8D57)
            kr0 = (key[0] + r * 0x9E3779B9) % (1 << 32)
            kr1 = (key[1] + r * 0xBB67AE85) % (1 << 32)
            ctr = [h1 ^ ctr[1] ^ kr0, l1, h0 ^ ctr[3] ^ kr1, l0]
        bits = torch.empty(grp.numel(), 8, dtype=torch.int64, device=_DEV)
        for j in range(4):
            bits[:, 2 * j] = ctr[j] % 65536
            bits[:, 2 * j + 1] = ctr[j] // 65536
        kept = bits.flatten()[:hi - lo] >= thr
        for o, k in zip(outs, names):
            v = s[k].flatten()[lo:hi].double()
            o[lo:hi] = torch.where(kept, v * 65536.0 / (65536 - thr), 0.0)
    return [o.view(s["x"].shape) for o in outs]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"norm": _exact_norm, "ffn": _exact_ffn, "dropout": _exact_dropout}[case["op"]](s, case)
