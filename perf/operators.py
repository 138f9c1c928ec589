"""The block-scaled FP8 operators as users call them, as timed cases.

Five kinds of case:

* ``quant``: ``fp8_quant_rows``, rows to e4m3 with an fp32 scale for each group of 128 columns (the attention output
  before its projection).
* ``norm``: ``fp8_norm_quant``, the residual's addition, the root-mean-square norm and the quantization in one pass,
  with the sum, and the normed rows too where a router or an EXL3 expert layer reads them.
* ``swiglu``: ``fp8_swiglu_quant``, gate and up to the quantized input of the down projection.
* ``linear``: ``fp8_linear``, the product with an e4m3 weight that has an fp32 scale for each 128 x 128 block, from
  16-bit rows (quantized inside) or from quantized rows.
* ``mlp``: the four together, as a decoder layer's second half runs them: norm, gate/up, SwiGLU, down.

Weights are e4m3 with block scales that differ by block; activations are N(0, 1) with a few loud columns.
"""

from __future__ import annotations

import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6          # of the norm
LEAST = 1e-10       # least largest magnitude of a group
TOP = 448.0         # the largest e4m3 value


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # one token's qkv projection, straight from the 16-bit rows
        {"name": "linear-rows-1", "kind": "linear", "m": 1, "k": 4096, "n": 6144, "rows": True, "bias": False,
         "dtype": "bfloat16"},
        # the down projection of a busy server's decode batch
        {"name": "linear-rows-24", "kind": "linear", "m": 24, "k": 14336, "n": 4096, "rows": True, "bias": False,
         "dtype": "bfloat16"},
        # a narrow latent projection (four and a half blocks wide) of a short ragged prompt, with a bias
        {"name": "linear-77", "kind": "linear", "m": 77, "k": 2048, "n": 576, "rows": False, "bias": True,
         "dtype": "float16"},
        # gate/up of a prefill chunk, compute bound
        {"name": "linear-2048", "kind": "linear", "m": 2048, "k": 4096, "n": 28672, "rows": False, "bias": False,
         "dtype": "bfloat16"},
        # one token's attention output: launch latency
        {"name": "quant-1", "kind": "quant", "m": 1, "k": 4096, "dtype": "bfloat16"},
        # a ragged prefill chunk of MLP width
        {"name": "quant-2049", "kind": "quant", "m": 2049, "k": 14336, "dtype": "bfloat16"},
        # one token between two layers
        {"name": "norm-1", "kind": "norm", "m": 1, "k": 4096, "residual": True, "rows": False, "dtype": "bfloat16"},
        # a prefill chunk before a sparse layer: the router and the EXL3 experts read the normed rows
        {"name": "norm-2048", "kind": "norm", "m": 2048, "k": 4096, "residual": True, "rows": True,
         "dtype": "bfloat16"},
        # a few tokens through a shared expert
        {"name": "swiglu-3", "kind": "swiglu", "m": 3, "n": 768, "limit": 0.0, "dtype": "bfloat16"},
        # a prefill chunk, with the clamp that some models set
        {"name": "swiglu-2048", "kind": "swiglu", "m": 2048, "n": 14336, "limit": 7.0, "dtype": "bfloat16"},
        # one token through a shared expert's whole MLP
        {"name": "mlp-1", "kind": "mlp", "m": 1, "k": 2048, "n": 768, "dtype": "bfloat16"},
        # a decode batch through a dense layer's whole MLP
        {"name": "mlp-40", "kind": "mlp", "m": 40, "k": 4096, "n": 14336, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("linear", "linear", "linear", "quant", "norm", "swiglu", "mlp"))
        case = {"kind": kind, "m": _log(rng, 1, 4096), "dtype": rng.choice(("float16", "bfloat16", "bfloat16"))}
        k = 16 * _log(rng, 16, 1024)  # rows of 256 to 16384, groups that end early among them
        if kind == "linear":
            case.update(k=k, n=_log(rng, 64, 28672), rows=rng.random() < 0.5, bias=rng.random() < 0.3)
        elif kind == "quant":
            case.update(k=k)
        elif kind == "norm":
            case.update(k=k, residual=rng.random() < 0.7, rows=rng.random() < 0.4)
        elif kind == "swiglu":
            case.update(n=k, limit=rng.choice((0.0, 0.0, 7.0)))
        else:
            case.update(m=_log(rng, 1, 512), k=16 * _log(rng, 32, 512), n=16 * _log(rng, 32, 1024))
        if _cost(case) <= most:
            return case


def _groups(k):
    return -(-k // 128)


def work(case):
    m, kind = case["m"], case["kind"]
    if kind == "linear":
        k, n = case["k"], case["n"]
        x = 2 * m * k if case["rows"] else m * k + 4 * m * _groups(k)
        w = n * k + 4 * _groups(n) * _groups(k) + (2 * n if case["bias"] else 0)
        return {"bytes": x + w + 2 * m * n, "flops": 2 * m * n * k}
    if kind == "quant":
        k = case["k"]
        return {"bytes": 3 * m * k + 4 * m * _groups(k), "flops": 4 * m * k}
    if kind == "norm":
        k = case["k"]
        extra = (4 if case["residual"] else 0) + (2 if case["rows"] else 0)
        return {"bytes": (3 + extra) * m * k + 2 * k + 4 * m * _groups(k), "flops": 9 * m * k}
    n = case["n"]
    if kind == "swiglu":
        return {"bytes": 5 * m * n + 4 * m * _groups(n), "flops": 10 * m * n}
    k = case["k"]  # mlp: two weights, the rows, the residual in and out, the result
    return {"bytes": 3 * n * k + 4 * (_groups(2 * n) * _groups(k) + _groups(k) * _groups(n)) + 2 * k + 8 * m * k,
            "flops": 6 * m * n * k}


# ------------------------------------------------------------------ inputs

def _rows(g, m, k, dtype):
    x = torch.randn((m, k), device="cuda", generator=g)
    loud = torch.rand((1, k), device="cuda", generator=g) < 0.005
    return (x * (1.0 + 7.0 * loud)).to(dtype)


def _weight(g, n, k):
    """An e4m3 weight and the scales of its 128 x 128 blocks, whose products are O(1) for N(0, 1) rows."""
    w = torch.randn((n, k), device="cuda", generator=g).mul_(100.0).clamp_(-TOP, TOP).to(torch.float8_e4m3fn)
    s = torch.randn((_groups(n), _groups(k)), device="cuda", generator=g).mul_(0.5).exp_()
    return w, s.mul_(0.01 / math.sqrt(k))


def prepare(case, seed):
    if own:
        _register()
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    m, kind, dt = case["m"], case["kind"], DTYPES[case["dtype"]]
    s = SimpleNamespace(kind=kind, bf16=dt == torch.bfloat16)
    if kind == "linear":
        k, n = case["k"], case["n"]
        s.x, s.xs = _rows(g, m, k, dt), None
        if not case["rows"]:
            s.x, s.xs = _quant(s.x.float())
        s.w, s.ws = _weight(g, n, k)
        s.bias = torch.randn((n,), device="cuda", generator=g).to(dt) if case["bias"] else None
    elif kind == "quant":
        s.x = _rows(g, m, case["k"], dt)
    elif kind == "norm":
        k = case["k"]
        s.x = _rows(g, m, k, dt)
        s.res = _rows(g, m, k, dt) * 2 if case["residual"] else None
        s.gain, s.rows = (1 + 0.2 * torch.randn((k,), device="cuda", generator=g)).to(dt), case["rows"]
    elif kind == "swiglu":
        s.x, s.limit = torch.randn((m, 2 * case["n"]), device="cuda", generator=g).mul_(2.5).to(dt), case["limit"]
    else:
        k, n = case["k"], case["n"]
        s.x, s.res = _rows(g, m, k, dt), _rows(g, m, k, dt) * 2
        s.gain = (1 + 0.2 * torch.randn((k,), device="cuda", generator=g)).to(dt)
        s.gu, s.down = _weight(g, 2 * n, k), _weight(g, k, n)
    return s


# ------------------------------------------------------------- the plain forms

def _grouped(x):
    """x [m, k] as groups of 128 columns, the last one filled with zeros."""
    m, k = x.shape
    pad = _groups(k) * 128 - k
    return (torch.cat((x, x.new_zeros((m, pad))), 1) if pad else x).view(m, -1, 128)


def _quant(x):
    """(e4m3 rows, fp32 scale of each group) of fp32 rows."""
    y = _grouped(x)
    most = y.abs().amax(-1).clamp(min=LEAST)
    t = y * TOP / most.unsqueeze(-1)  # exact ties of 16-bit rows stay ties, which y / scale would not keep
    return t.view(x.shape[0], -1)[:, :x.shape[1]].to(torch.float8_e4m3fn), most / TOP


def _norm(x, res, gain):
    h = x.float() if res is None else x.float() + res.float()
    return h, h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * gain.float()


def _swiglu(x, limit):
    a, b = x.float().chunk(2, -1)
    if limit:
        a, b = a.clamp(max=limit), b.clamp(-limit, limit)
    return a / (1 + torch.exp(-a)) * b


def _linear(q, s, w, ws, bias, dtype):
    x = (_grouped(q.float()) * s.unsqueeze(-1)).view(q.shape[0], -1)[:, :q.shape[1]]
    n, k = w.shape
    y = x @ (w.float() * ws.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).t()
    return (y if bias is None else y + bias.float()).to(dtype)


def _plain(s):
    if s.kind == "linear":
        q, xs = _quant(s.x.float()) if s.xs is None else (s.x, s.xs)
        return _linear(q, xs, s.w, s.ws, s.bias, torch.bfloat16 if s.bf16 else torch.float16)
    if s.kind == "quant":
        return _quant(s.x.float())
    if s.kind == "norm":
        h, y = _norm(s.x, s.res, s.gain)
        more = [h.to(s.x.dtype)] if s.res is not None else []
        return [*_quant(y), *more, *([y.to(s.x.dtype)] if s.rows else [])]
    if s.kind == "swiglu":
        return _quant(_swiglu(s.x, s.limit))
    h, y = _norm(s.x, s.res, s.gain)
    gu = _linear(*_quant(y), *s.gu, None, s.x.dtype)
    return _linear(*_quant(_swiglu(gu, 0.0)), *s.down, None, s.x.dtype), h.to(s.x.dtype)


# ------------------------------------------------------- the framework's calls

def _register():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang-exl3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sglang_exl3.ops import register_custom_ops

    register_custom_ops()


def _calls(s):
    o = torch.ops.sglang_exl3
    if s.kind == "linear":
        return o.fp8_linear(s.x, s.w, s.ws, s.xs, s.bias, s.bf16)
    if s.kind == "quant":
        return o.fp8_quant_rows(s.x)
    if s.kind == "norm":
        return o.fp8_norm_quant(s.x, s.gain, EPS, s.res, s.rows)
    if s.kind == "swiglu":
        return o.fp8_swiglu_quant(s.x, s.limit)
    q, xs, h = o.fp8_norm_quant(s.x, s.gain, EPS, s.res, False)
    gu = o.fp8_linear(q, *s.gu, xs, None, s.bf16)
    q, xs = o.fp8_swiglu_quant(gu, 0.0)
    return o.fp8_linear(q, *s.down, xs, None, s.bf16), h


def run(state):
    return _calls(state) if own else _plain(state)


# --------------------------------------------------------------- in 64 bits

def _near(v):
    """The e4m3 values nearest to v (float64, at most 448 in size), ties to the even one: steps of 2^(e - 3) from
    2^e on, and of 2^-9 below 2^-6."""
    step = torch.exp2(torch.frexp(v).exponent.sub(1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def _exact_groups(v):
    """(v over its groups' scales, the scales), each group of 128 columns, both in 64 bits."""
    out, scales = torch.empty_like(v), []
    for c in range(0, v.shape[1], 128):
        part = v[:, c:c + 128]
        most = part.abs().amax(1, keepdim=True).clamp(min=LEAST)
        out[:, c:c + 128] = part * TOP / most
        scales.append(most / TOP)
    return out, torch.cat(scales, 1)


def _spread(s, k):
    """A scale for each column from one for each group of 128."""
    return s[:, torch.arange(k, device=s.device) // 128]


def _exact_linear(v, w, ws):
    """The product of quantized v (float64) with the weight."""
    n, k = w.shape
    t, s = v
    x = t * _spread(s.double(), k)
    return x @ (w.double() * _spread(ws.double().t(), n).t()[:, torch.arange(k, device=w.device) // 128]).t()


def _exact_quant(v):
    t, s = _exact_groups(v)
    return _near(t), s


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        v = _exact_quant(s.x.double()) if case["rows"] else (s.x.double(), s.xs)
        y = _exact_linear(v, s.w, s.ws)
        return y + s.bias.double() if case["bias"] else y
    if kind == "quant":
        return _exact_groups(s.x.double())
    if kind == "swiglu":
        a, b = s.x.double().split(case["n"], 1)
        if case["limit"]:
            a, b = torch.clamp(a, max=case["limit"]), torch.clamp(b, -case["limit"], case["limit"])
        return _exact_groups(a * torch.sigmoid(a) * b)
    h = s.x.double() + s.res.double() if s.res is not None else s.x.double()
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS) * s.gain.double()
    if kind == "norm":
        return [*_exact_groups(y), *([h] if case["residual"] else []), *([y] if case["rows"] else [])]
    gu = _exact_linear(_exact_quant(y), *s.gu).to(s.x.dtype).double()
    a, b = gu.split(case["n"], 1)
    return _exact_linear(_exact_quant(a * torch.sigmoid(a) * b), *s.down), h
