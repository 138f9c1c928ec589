"""The block-scaled FP8 operators in 64 bits, and the errors that fp32 arithmetic may add."""

from __future__ import annotations

import torch

U = 2.0 ** -24  # half a step of fp32, relative


def near(v: torch.Tensor) -> torch.Tensor:
    """v (float64, at most 448 in size) rounded to e4m3, ties to even."""
    step = torch.exp2(torch.frexp(v).exponent.sub(1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def half_step(v: torch.Tensor) -> torch.Tensor:
    """Half the distance of e4m3 neighbours around v."""
    return torch.exp2(torch.frexp(v).exponent.sub(1).clamp(min=-6).double() - 4)


def grouped(v: torch.Tensor) -> torch.Tensor:
    k = v.shape[-1]
    return torch.nn.functional.pad(v, (0, -k % 128)).reshape(*v.shape[:-1], -1, 128)


def spread(s: torch.Tensor, k: int) -> torch.Tensor:
    return s.repeat_interleave(128, -1)[..., :k]


def quant64(v: torch.Tensor):
    """(448 v / a, a / 448) of each group in float64, a = max(max |v|, fp32(1e-10))."""
    v = v.double()
    a = grouped(v).abs().amax(-1).clamp(min=float(torch.tensor(1e-10)))
    return v * 448 / spread(a, v.shape[-1]), a / 448


def norm64(x, weight, eps, residual=None):
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / (h.square().mean(-1, keepdim=True) + float(torch.tensor(eps))).sqrt() * weight.double()


def swiglu64(x, limit=0.0):
    g, u = x.double().chunk(2, -1)
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(g) * u


def weight64(w, ws):
    n, k = w.shape
    return w.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def linear64(q, s, w, ws, bias=None):
    """(the product, the sum of its terms' sizes) of quantized rows in float64."""
    x, wd = q.double() * spread(s.double(), q.shape[-1]), weight64(w, ws)
    y, size = x @ wd.t(), x.abs() @ wd.abs().t()
    return (y, size) if bias is None else (y + bias.double(), size + bias.double().abs())


def make_weight(n, k, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn((n, k), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = torch.exp(torch.randn((-(-n // 128), -(-k // 128)), generator=g)) / (100 * k ** 0.5)
    return w.to(device), ws.to(device)


def make_rows(m, k, seed, dtype=torch.bfloat16, device="cuda"):
    g = torch.Generator().manual_seed(seed + 1000)
    x = torch.randn((m, k), generator=g) * torch.exp(torch.randn((m, 1), generator=g))
    x[:, torch.rand(k, generator=g) < 0.01] *= 16
    return x.to(dtype).to(device)


def check_quant(q, s, v64, slack, what=""):
    """(q, s) against the fp64 values v64 that they quantize, known to the relative error `slack` (of the largest
    of the group): the scale to slack and its own rounding, q to half an e4m3 step and the error of the quotient."""
    t, s64 = quant64(v64)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and q.shape == v64.shape
    assert s.shape == s64.shape, what
    assert float(((s.double() - s64) / s64).abs().max()) <= slack + 2 * U, what
    # a value and the largest one are each off by slack, and three roundings follow
    bound = half_step(t) * (1 + 2.0 ** -20) + (2 * slack + 3 * U) * 448
    assert bool(((q.double() - t).abs() <= bound).all()), what


def largest_products(x, wd):
    """The largest |x[m, j] w[n, j]| of each block of 128 columns, summed over the blocks."""
    wb = grouped(wd.float()).abs()
    return torch.stack([(grouped(r).abs() * wb).amax(-1).sum(-1) for r in x.float()]).double()


def check_product(y, q, s, w, ws, bias=None, what=""):
    """y against the float64 product of the same quantized rows.

    The matrix unit adds e4m3 products in groups of 16: it aligns them to the largest exponent of the group and drops
    what lies 13 bits below it, then adds the group in fp32.  (Measured with one large product, its negative and one
    small one: for 2^(2a) the smallest that survives in the group is 2^(2a - 13); a term never loses more than that.)
    So a block of 128 columns is off by at most 8 groups x 15 others x 2^-13 of its largest product.  The groups' sum
    and the blocks' in fp32 add at most one U of the sum of sizes for each of 8 + 1 steps a block, twice that where
    bits are dropped and not rounded; the scales' product, its use and the bias are 3 U more; then half a step of y.

    That is the worst case.  The dropped parts have both signs, and in the norm they are 2e-5 of y for random
    operands, 2e-4 with a column 16 times as loud; half a step of y's type is at most 1 / sqrt(3) of itself there."""
    wd = weight64(w, ws)
    y64, size = linear64(q, s, w, ws, bias)
    eps = torch.finfo(y.dtype).eps / 2
    blocks = -(-q.shape[-1] // 128)
    fp32 = 120 * 2.0 ** -13 * largest_products(q.double() * spread(s.double(), q.shape[-1]), wd)
    fp32 += (2 * 9 * blocks + 8) * U * size
    bound = fp32 + eps * (y64.abs() + fp32) + float(torch.finfo(y.dtype).smallest_normal) * eps * 2
    err = y.double() - y64
    far = float((err.abs() - bound).max())
    assert far <= 0, f"{what}: {far:.3g} beyond the bound"
    if y.numel() >= 1024:
        rel = float(err.norm() / y64.norm())
        assert rel <= eps / 3 ** 0.5 + 2e-4, f"{what}: relative error {rel:.3g}"
