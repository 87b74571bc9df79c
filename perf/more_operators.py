"""The operators of an mHC model's attention sublayer, between the projections
of its input: rotary positions and attention, as programs that train or serve
the model run them.

A case is one pass, inputs resident on the GPU: a forward call (``train``
false: serving) or a forward and its backward (``train`` true).  With ``own``
false, ``run`` computes the formulas with elementary torch operations in 32
bits (the rotation's angles in 64); with ``own`` true it calls
``FlagOS_mhc.sublayer``.  ``exact`` is the same in 64 bits, written apart.

Keys of a case:
  op      "rotary", "attention" (packed sequences) or "decode" (the attention
          of the last tokens over a cache of fixed size)
  H, Hk   heads of the queries, and of the keys and values
  d       head width
  dtype   of the activations
  train   forward and backward instead of the forward alone
  T, B    (rotary, attention) tokens and sequences; (decode) B sequences of S new tokens
  pad     (attention) rows of the buffers behind the last sequence
  empty   (attention, decode) the second sequence has no tokens (keys)
  L       (decode) rows of a sequence's cache; the sequences use between half of them and all
  causal  (attention) a query sees the keys up to its own place, or all
  r       (rotary) rotated width, the first r of d
  layout  (rotary) "half" (pairs i, i + r/2) or "interleaved" (pairs 2i, 2i + 1)
  scaling (rotary) None, "linear", "ntk" or "yarn", by factor 8 from 8192 positions
  far     (rotary) the first position: prompts start at 0, decoding goes on from a long context
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_DEV = "cuda"
_BASE, _FACTOR, _LENGTH = 10000.0, 8.0, 8192


def _named(name, c):
    if name:
        c["name"] = name
    return c


def _rot(name, T, H, Hk, d, r=None, dtype="bf16", layout="half", scaling=None, far=0, B=1, train=False):
    return _named(name, dict(op="rotary", T=T, H=H, Hk=Hk, d=d, r=r or d, dtype=dtype, layout=layout,
                             scaling=scaling, far=far, B=B, train=train))


def _att(name, T, B, H, Hk, d, dtype="bf16", causal=True, pad=0, empty=False, train=False):
    return _named(name, dict(op="attention", T=T, B=B, H=H, Hk=Hk, d=d, dtype=dtype, causal=causal, pad=pad,
                             empty=empty, train=train))


def _dec(name, B, S, L, H, Hk, d, dtype="bf16", empty=False):
    return _named(name, dict(op="decode", B=B, S=S, L=L, H=H, Hk=Hk, d=d, dtype=dtype, empty=empty, train=False))


def listed():
    return [
        # one token of each of 64 sequences of a decoding loop, far into their contexts
        _rot("rotary_decode", 64, 32, 8, 128, scaling="yarn", far=60000),
        # a prompt of odd length in fp16, half of the head rotated, neighbours as pairs
        _rot("rotary_prefill_part_f16", 2049, 16, 16, 80, 40, "f16", "interleaved", "ntk"),
        # the benchmark's batch: 65536 tokens in 16 packed sequences at width 56 x 128, forward and backward
        _rot("rotary_train_large", 65536, 56, 8, 128, B=16, train=True),
        # one token over one long context: a single sequence of a decoding loop
        _dec("decode_b1", 1, 1, 32768, 32, 8, 128),
        # a decoding batch of 64 sequences of different lengths
        _dec("decode_b64", 64, 1, 8192, 32, 8, 128),
        # a short prompt in fp16, odd lengths, a head that is no power of two wide
        _att("prefill_odd_f16", 777, 3, 16, 4, 80, "f16"),
        # one long prompt
        _att("prefill_long", 32768, 1, 32, 8, 128),
        # a small fp32 model's training step
        _att("train_f32", 1021, 2, 8, 8, 64, "f32", train=True),
        # a middle-sized model's training step over packed documents, an empty one and padding among them
        _att("train_packed", 8192, 9, 16, 4, 64, pad=57, empty=True, train=True),
        # an encoder's step: every token sees its whole document
        _att("train_all", 4099, 5, 32, 8, 128, causal=False, train=True),
        # a large model's training step at width 56 x 128, one sequence
        _att("train_large", 16384, 1, 56, 8, 128, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(4, 4), (8, 8), (8, 1), (12, 4), (16, 4), (16, 16), (32, 8), (40, 8), (56, 8)]


def draw(rng):
    op = rng.choice(["rotary", "rotary", "attention", "attention", "attention", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    H, Hk = rng.choice(_HEADS)
    d = rng.choice([64, 128, 128, 128, 80, 96, 192, 256, rng.randrange(16, 200, 2)])
    if op == "rotary":
        T = _log_int(rng, 1, 65536 if dtype != "f32" else 16384)
        r = d if rng.random() < 0.6 else max(2, d // rng.choice([2, 4]) // 2 * 2)
        # at most the largest listed case's rows
        return _rot(None, max(1, min(T, 65536 * 64 * 128 // (2 * (H + Hk) * d))), H, Hk, d, r, dtype, rng.choice(["half", "interleaved"]),
                    rng.choice([None, "linear", "ntk", "yarn"]), rng.choice([0, _log_int(rng, 1, 500000)]),
                    1, rng.random() < 0.5)
    if dtype == "f32":
        d = min(d, 128)
    if op == "decode":
        B = _log_int(rng, 1, 64)
        # at most the cache of the largest listed case
        L = _log_int(rng, 16, min(32768, 64 * 8192 * 8 * 128 * 2 // (B * Hk * d * _SIZE[dtype])))
        return _dec(None, B, rng.choice([1, 1, 1, 2, 5]), L, H, Hk, d, dtype, rng.random() < 0.2)
    if d > 128:
        H, Hk = H // 2, max(1, Hk // 2)
        H -= H % Hk
    T = _log_int(rng, 1, 16384 if dtype != "f32" else 2048)
    B = rng.randint(1, max(1, min(T // 2, 16)))
    return _att(None, T, B, H, Hk, d, dtype, rng.random() < 0.8, rng.choice([0, 0, rng.randint(1, 300)]),
                rng.random() < 0.3, rng.random() < 0.6)


# ---- inputs -------------------------------------------------------------------

def _lengths(case):
    """Tokens of each packed sequence: different ones, T in all."""
    T, B = case["T"], case["B"]
    if B == 1:
        return [T]
    w = [0.25 + ((b + 1) * 0.6180339887498949) % 1.0 for b in range(B)]
    if case.get("empty"):
        w[1] = 0.0
    n = [int(T * v / sum(w)) for v in w]
    n[-1] += T - sum(n)
    return n


def _used(case):
    """Rows of each sequence's cache that hold keys."""
    L, B = case["L"], case["B"]
    n = [L if b == 0 else L - int(L // 2 * ((b * 0.6180339887498949) % 1.0)) for b in range(B)]
    if case["empty"] and B > 1:
        n[1] = 0
    return n


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _inputs(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]
    H, Hk, d = case["H"], case["Hk"], case["d"]

    def heads(*lead):
        # projections' results: columns of different sizes
        col = torch.exp(0.3 * torch.randn(lead[-1], d, device=_DEV, generator=g))
        return torch.randn(*lead, d, device=_DEV, generator=g).mul_(col).to(dt)

    s = {}
    if case["op"] == "decode":
        B, S, L = case["B"], case["S"], case["L"]
        s["q"], s["k"], s["v"] = heads(B, S, H), heads(B, L, Hk), heads(B, L, Hk)
        s["used"] = torch.tensor(_used(case), dtype=torch.int32, device=_DEV)
        return s
    rows = case["T"] + case.get("pad", 0)
    starts = _starts(_lengths(case))
    s["q"], s["k"] = heads(rows, H), heads(rows, Hk)
    if case["train"]:
        s["gq"] = torch.randn(rows, H, d, device=_DEV, generator=g).to(dt)
    if case["op"] == "rotary":
        if case["train"]:
            s["gk"] = torch.randn(rows, Hk, d, device=_DEV, generator=g).to(dt)
        t = torch.arange(rows, device=_DEV)
        at = torch.tensor(starts, device=_DEV)
        s["positions"] = (t - at[torch.searchsorted(at, t, right=True) - 1] + case["far"]).to(torch.int32)
        return s
    s["v"] = heads(rows, Hk)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=_DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if case["op"] == "rotary":
        if own:
            s["freqs"], s["amplitude"] = _sublayer().rotary_frequencies(
                case["r"], _BASE, scaling=case["scaling"], factor=_FACTOR, original_length=_LENGTH, device=_DEV)
        else:
            s["freqs"], s["amplitude"] = _plain_frequencies(case)
    return s


# ---- the plain form ---------------------------------------------------------------

def _plain_frequencies(c):
    """Radians a position of each pair, in 64 bits, and the factor on the result."""
    r, kind = c["r"], c["scaling"]
    base = _BASE * _FACTOR ** (r / (r - 2)) if kind == "ntk" and r > 2 else _BASE
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device=_DEV) / r)
    if kind == "linear":
        return f / _FACTOR, 1.0
    if kind == "yarn":
        # pairs that turn often over the original length stay, those that do not even turn once are stretched
        keep = ((_LENGTH * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        return f * keep + f / _FACTOR * (1.0 - keep), 0.1 * math.log(_FACTOR) + 1.0
    return f, 1.0


def _plain_rotate(x, cos, sin, r, layout):
    xf = x.float()
    out = xf.clone()
    if layout == "half":
        a, b = xf[..., :r // 2], xf[..., r // 2:r]
        out[..., :r // 2] = a * cos - b * sin
        out[..., r // 2:r] = a * sin + b * cos
    else:
        a, b = xf[..., 0:r:2], xf[..., 1:r:2]
        out[..., 0:r:2] = a * cos - b * sin
        out[..., 1:r:2] = a * sin + b * cos
    return out.to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["freqs"]
    cos = (torch.cos(angle) * s["amplitude"]).float()[:, None, :]
    sin = (torch.sin(angle) * s["amplitude"]).float()[:, None, :]
    out = [_plain_rotate(s[n], cos, sin, c["r"], c["layout"]) for n in ("q", "k")]
    if c["train"]:
        out += [_plain_rotate(s[n], cos, -sin, c["r"], c["layout"]) for n in ("gq", "gk")]
    return out


def _plain_softmax(score):
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0.0, 1.0, total)


def _plain_attention(s):
    c = s["case"]
    H, Hk, d = c["H"], c["Hk"], c["d"]
    G, scale = H // Hk, c["d"] ** -0.5
    dt, train = s["q"].dtype, c["train"]
    out = torch.zeros_like(s["q"])
    grads = [torch.zeros_like(s[n]) for n in ("q", "k", "v")] if train else []
    lo = 0
    for n in _lengths(c):
        rows = slice(lo, lo + n)
        lo += n
        if n == 0:
            continue
        # as many heads at a time as 2^30 scores hold
        step = max(1, min(Hk, (1 << 30) // (n * n * G)))
        groups = max(1, min(G, (1 << 30) // (n * n))) if step == 1 else G
        hidden = torch.ones(n, n, dtype=torch.bool, device=_DEV).triu(1) if c["causal"] else None
        for h in range(0, Hk, step):
            kv = slice(h, min(h + step, Hk))
            m = kv.stop - kv.start
            k = s["k"][rows, kv].float().transpose(0, 1).contiguous()  # (m, n, d)
            v = s["v"][rows, kv].float().transpose(0, 1).contiguous()
            gk, gv = torch.zeros_like(k), torch.zeros_like(v)
            for g in range(0, G, groups):
                e = min(g + groups, G)

                def take(t):  # (m, heads * n, d)
                    return (t[rows].float().view(n, Hk, G, d)[:, kv, g:e].permute(1, 2, 0, 3)
                            .reshape(m, (e - g) * n, d).contiguous())

                def put(t, val):
                    t[rows].view(n, Hk, G, d)[:, kv, g:e] = val.view(m, e - g, n, d).permute(2, 0, 1, 3).to(dt)

                q = take(s["q"])
                score = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(scale)
                if hidden is not None:
                    score.view(m, e - g, n, n).masked_fill_(hidden, -math.inf)
                p = _plain_softmax(score)
                del score
                o = torch.bmm(p, v)
                put(out, o)
                if not train:
                    continue
                go = take(s["gq"])
                gv += torch.bmm(p.transpose(1, 2).contiguous(), go)
                ds = torch.bmm(go, v.transpose(1, 2).contiguous()).sub_((go * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                del p
                put(grads[0], torch.bmm(ds, k))
                gk += torch.bmm(ds.transpose(1, 2).contiguous(), q)
            if train:
                grads[1][rows, kv] = gk.transpose(0, 1).to(dt)
                grads[2][rows, kv] = gv.transpose(0, 1).to(dt)
    return [out, *grads]


def _plain_decode(s):
    c = s["case"]
    B, S, L, H, Hk, d = (c[n] for n in ("B", "S", "L", "H", "Hk", "d"))
    G = H // Hk
    used = s["used"].long()
    # row j of the cache is seen by new token i of the last S
    at = torch.arange(L, device=_DEV)
    seen = at[None, None, :] <= (used[:, None, None] - S + torch.arange(S, device=_DEV)[None, :, None])
    seen &= (at < used[:, None])[:, None, :]
    out = torch.empty_like(s["q"])
    step = max(1, (1 << 29) // (L * Hk * d))
    for b in range(0, B, step):
        e = min(b + step, B)
        q = s["q"][b:e].float().view(e - b, S, Hk, G, d).permute(0, 2, 3, 1, 4).reshape(-1, G * S, d).contiguous()
        kt = s["k"][b:e].float().permute(0, 2, 3, 1).reshape(-1, d, L).contiguous()
        score = torch.bmm(q, kt).mul_(d ** -0.5).view(e - b, Hk, G, S, L)
        score.masked_fill_(~seen[b:e, None, None], -math.inf)
        v = s["v"][b:e].float().transpose(1, 2).reshape(-1, L, d).contiguous()
        o = torch.bmm(_plain_softmax(score).view(-1, G * S, L), v)
        out[b:e] = o.view(e - b, Hk, G, S, d).permute(0, 3, 1, 2, 4).reshape(e - b, S, H, d).to(out.dtype)
    return [out]


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


def _own_rotary(s):
    c, lib = s["case"], _sublayer()
    kw = dict(layout=c["layout"], amplitude=s["amplitude"])
    out = [*lib.rotary(s["q"], s["k"], s["freqs"], s["positions"], **kw)]
    if c["train"]:
        out += lib.rotary_backward(s["gq"], s["gk"], s["freqs"], s["positions"], **kw)
    return out


def _own_attention(s):
    c, lib = s["case"], _sublayer()
    if not c["train"]:
        return [lib.attention(s["q"], s["k"], s["v"], s["starts"], causal=c["causal"])["out"]]
    f = lib.attention(s["q"], s["k"], s["v"], s["starts"], causal=c["causal"], need_backward=True)
    return [f["out"], *lib.attention_backward(s["gq"], s["q"], s["k"], s["v"], f["out"], f["lse"], s["starts"],
                                              causal=c["causal"])]


def _own_decode(s):
    return [_sublayer().attention(s["q"], s["k"], s["v"], lengths_k=s["used"])["out"]]


_PLAIN = {"rotary": _plain_rotary, "attention": _plain_attention, "decode": _plain_decode}
_OWN = {"rotary": _own_rotary, "attention": _own_attention, "decode": _own_decode}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


# ---- floors ------------------------------------------------------------------------

def work(case):
    H, Hk, d, e = case["H"], case["Hk"], case["d"], _SIZE[case["dtype"]]
    if case["op"] == "rotary":
        passes = 2 if case["train"] else 1
        n = passes * case["T"] * (H + Hk)
        # q and k read and written, the positions; six operations a rotated pair
        return {"bytes": 2 * n * d * e + 4 * case["T"], "flops": 3 * n * case["r"]}
    if case["op"] == "decode":
        used, S = _used(case), case["S"]
        pairs = sum(max(0, n - S + i + 1) for n in used for i in range(S))
        return {"bytes": (2 * case["B"] * S * H + 2 * sum(used) * Hk) * d * e, "flops": 4 * pairs * H * d}
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
    q, kv = case["T"] * H * d * e, case["T"] * Hk * d * e
    if not case["train"]:
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * H * d}
    # two products forward; the scores again and four backward
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * H * d}


# ---- the definition in 64 bits -----------------------------------------------------------

def _exact_rotary(s, case):
    r, half = case["r"], case["r"] // 2
    L, factor = float(_LENGTH), _FACTOR
    rows = []
    for i in range(half):
        w = _BASE ** (-2.0 * i / r)
        if case["scaling"] == "linear":
            w /= factor
        elif case["scaling"] == "ntk" and r > 2:
            w = (_BASE * factor ** (r / (r - 2.0))) ** (-2.0 * i / r)
        elif case["scaling"] == "yarn":
            turns = L * w / (2.0 * math.pi)
            part = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            w = (1.0 - part) * w / factor + part * w
        rows.append(w)
    amp = 1.0 + 0.1 * math.log(factor) if case["scaling"] == "yarn" else 1.0
    w = torch.tensor(rows, dtype=torch.float64, device=_DEV)
    first = torch.arange(half, device=_DEV)
    a, b = (first, first + half) if case["layout"] == "half" else (2 * first, 2 * first + 1)
    outs = []
    for name, sign in (("q", 1.0), ("k", 1.0), ("gq", -1.0), ("gk", -1.0)):
        if name not in s:
            continue
        y = s[name].to(torch.float64)
        for lo in range(0, y.shape[0], 4096):
            blk = y[lo:lo + 4096]
            turn = torch.polar(torch.full((blk.shape[0], half), amp, dtype=torch.float64, device=_DEV),
                               sign * torch.outer(s["positions"][lo:lo + 4096].double(), w))[:, None]
            z = torch.complex(blk[..., a], blk[..., b]) * turn
            blk[..., a], blk[..., b] = z.real, z.imag
        outs.append(y)
    return outs


def _exact_head(q, k, v, go, scale, offset):
    """One head's output, and gradients if go: query i sees keys up to i + offset (None: all)."""
    n, L = q.shape[0], k.shape[0]
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    kt, vt = k.t().contiguous(), v.t().contiguous()
    for lo in range(0, n, 8192):
        hi = min(lo + 8192, n)
        z = torch.mm(q[lo:hi], kt) * scale
        if offset is not None:
            i = torch.arange(lo, hi, device=_DEV)[:, None]
            z = torch.where(torch.arange(L, device=_DEV)[None, :] <= i + offset, z, -math.inf)
        norm = torch.logsumexp(z, 1, keepdim=True)
        w = torch.exp(z - torch.where(norm == -math.inf, 0.0, norm))
        del z
        out[lo:hi] = torch.mm(w, v)
        if go is None:
            continue
        d = go[lo:hi]
        dv += torch.mm(w.t().contiguous(), d)
        t = torch.mm(d, vt)
        t = w * (t - (w * t).sum(1, keepdim=True)) * scale
        dq[lo:hi] = torch.mm(t, k)
        dk += torch.mm(t.t().contiguous(), q[lo:hi])
    return out, dq, dk, dv


def _exact_attention(s, case):
    H, Hk = case["H"], case["Hk"]
    scale = 1.0 / math.sqrt(case["d"])
    res = [torch.zeros(s[n].shape, dtype=torch.float64, device=_DEV) for n in ("q", "q", "k", "v")]
    for lo, hi in zip(_starts(_lengths(case)), _starts(_lengths(case))[1:]):
        if lo == hi:
            continue
        for h in range(H):
            c = h * Hk // H
            q, k, v = s["q"][lo:hi, h].double(), s["k"][lo:hi, c].double(), s["v"][lo:hi, c].double()
            go = s["gq"][lo:hi, h].double() if case["train"] else None
            o, dq, dk, dv = _exact_head(q, k, v, go, scale, 0 if case["causal"] else None)
            res[0][lo:hi, h], res[1][lo:hi, h] = o, dq
            res[2][lo:hi, c] += dk
            res[3][lo:hi, c] += dv
    return res if case["train"] else res[:1]


def _exact_decode(s, case):
    H, Hk, S = case["H"], case["Hk"], case["S"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    for b, n in enumerate(_used(case)):
        for c in range(Hk if n else 0):
            k, v = s["k"][b, :n, c].double(), s["v"][b, :n, c].double()
            for h in range(c * (H // Hk), (c + 1) * (H // Hk)):
                out[b, :, h] = _exact_head(s["q"][b, :, h].double(), k, v, None, 1.0 / math.sqrt(case["d"]), n - S)[0]
    return [out]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "decode": _exact_decode}[case["op"]](s, case)
