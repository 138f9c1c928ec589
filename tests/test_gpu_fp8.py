"""The block-scaled FP8 operators on the GPU against 64-bit arithmetic, at the sizes and values where they can go wrong."""

import pytest
import torch

from fp8_util import U, check_product, check_quant, half_step, make_rows, make_weight, near, norm64, quant64, swiglu64
from sglang_exl3 import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _registered():
    ops.register_custom_ops()


def op():
    return torch.ops.sglang_exl3


# ------------------------------------------------------------------ quantized rows

@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_16_bit_number(dtype):
    """Every finite number, each in a group whose largest is 1.75 (scale 2^-8: ties are common) or 1 or its own size."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    v = bits[torch.isfinite(bits)]
    for top in (1.75, 1.0, 0.8125, 61440.0):
        t = torch.tensor(top).to(dtype)
        vals = v[v.abs() <= t]
        vals = torch.cat((vals, vals.new_zeros(-len(vals) % 127))).view(-1, 127)
        x = torch.cat((vals, t.expand(len(vals), 1)), 1).cuda()
        q, s = op().fp8_quant_rows(x)
        t64, s64 = quant64(x)
        assert torch.equal(s.double(), s64.float().double())
        assert torch.equal(q.double(), near(t64)), top


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (3, 144), (5, 256), (2, 2064), (129, 4096), (33, 14336), (1, 65536)])
def test_quant_rows(m, k, dtype):
    x = make_rows(m, k, m + k, dtype)
    q, s = op().fp8_quant_rows(x)
    t, s64 = quant64(x)
    assert torch.equal(s, s64.float()) and torch.equal(q.double(), near(t))


def test_quant_strides_shapes_and_empty():
    x = make_rows(6, 512, 1)
    want = op().fp8_quant_rows(x)
    wide = torch.full((6, 1040), float("nan"), dtype=BF, device="cuda")
    wide[:, 16:528] = x
    odd = torch.empty(6 * 512 + 1, dtype=BF, device="cuda")
    odd[1:] = x.reshape(-1)
    cases = [wide[:, 16:528], odd[1:].view(6, 512), x.t().contiguous().t(), x.view(2, 3, 512)]
    off = torch.full((6, 1037), float("nan"), dtype=BF, device="cuda")  # rows at odd strides
    off[:, 3:515] = x
    cases += [off[:, 3:515]]
    for c in cases:
        q, s = op().fp8_quant_rows(c)
        assert q.shape == c.shape and s.shape == (*c.shape[:-1], 4)
        assert torch.equal(q.view(6, 512).float(), want[0].float()) and torch.equal(s.view(6, 4), want[1])
    q, s = op().fp8_quant_rows(x[0])
    assert torch.equal(q.float(), want[0][0].float()) and s.shape == (4,)
    q, s = op().fp8_quant_rows(x[:1].expand(4, 512))
    assert torch.equal(q.float(), want[0][:1].float().expand(4, 512))
    q, s = op().fp8_quant_rows(x[:0])
    assert q.shape == (0, 512) and s.shape == (0, 4)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quant_zeros_infinities_and_nan(dtype):
    x = make_rows(8, 384, 3, dtype)
    x[0] = 0
    x[1, :128] = -0.0
    x[2, 130] = float("inf")
    x[3, 140] = float("-inf")
    x[4, 300] = float("nan")
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).tiny / 4  # subnormal numbers
    q, s = op().fp8_quant_rows(x)
    f = q.float()
    assert (f[0] == 0).all() and torch.equal(s[0], quant64(x[0])[1].float())
    assert (f[1, :128] == 0).all()
    for r, at in ((2, 130), (3, 140)):
        assert s[r, 1] == float("inf") and f[r, at].isnan()
        rest = torch.cat((f[r, 128:at], f[r, at + 1:256]))
        assert (rest == 0).all() and s[r, [0, 2]].isfinite().all() and f[r, :128].isfinite().all()
    assert s[4, 2].isnan() and f[4, 256:].isnan().all() and f[4, :256].isfinite().all()
    for r in (5, 6):
        t, s64 = quant64(x[r])
        assert torch.equal(s[r], s64.float()) and torch.equal(f[r].double(), near(t))


# -------------------------------------------------------------------------- norm

def norm_slack(cols):
    """Relative error of a normed value in fp32: the sum of squares, by chains of at most 32 and a tree of at most
    6 + 16, the squares, the mean, eps, root, quotient and two products; half of what enters the root comes out."""
    return ((32 + 22 + 4) / 2 + 6) * U


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (3, 144), (2, 1008), (130, 2048), (7, 4096), (3, 5120), (2, 16400),
                                 (2, 32768)])
@pytest.mark.parametrize("residual,rows", [(False, False), (True, False), (True, True), (False, True)])
def test_norm_quant(m, k, dtype, residual, rows):
    x = make_rows(m, k, k, dtype)
    res = make_rows(m, k, k + 1, dtype) if residual else None
    w = (1 + 0.3 * torch.randn(k, generator=torch.Generator().manual_seed(k))).to(dtype).cuda()
    out = op().fp8_norm_quant(x, w, 1e-5, res, rows)
    assert len(out) == 2 + residual + rows
    h, y = norm64(x, w, 1e-5, res)
    check_quant(out[0], out[1], y, norm_slack(k) + 2 * U, f"{m} x {k}")
    if residual:  # the fp32 sum of two 16-bit numbers, rounded once more
        assert torch.equal(out[2], (x.float() + res.float()).to(dtype))
    if rows:
        eps = torch.finfo(dtype).eps / 2
        err = (out[-1].double() - y).abs()
        assert bool((err <= (eps * 1.001 + norm_slack(k)) * y.abs() + torch.finfo(dtype).smallest_normal * eps * 2).all())


def test_norm_strides_zeros_and_nan():
    x, res = make_rows(5, 256, 9), make_rows(5, 256, 10)
    w = torch.ones(256, dtype=BF, device="cuda")
    want = op().fp8_norm_quant(x, w, 1e-6, res, True)
    wide = torch.full((5, 776), float("nan"), dtype=BF, device="cuda")
    wide[:, 8:264], wide[:, 512:768] = x, res
    got = op().fp8_norm_quant(wide[:, 8:264], w, 1e-6, wide[:, 512:768], True)
    odd = torch.ones(257, dtype=BF, device="cuda")[1:]  # a weight that is not 16-byte aligned
    for a, b, c in zip(want, got, op().fp8_norm_quant(x.view(1, 5, 256), odd, 1e-6, res.view(1, 5, 256), True)):
        assert torch.equal(a.float(), b.float()) and torch.equal(a.float(), c.float().view(a.shape))
    # a row of zeros stays zeros, also without eps; a NaN or an infinity stays in its row
    x[0], res[0] = 0, 0
    x[2, 7], x[3, 200] = float("nan"), float("inf")
    q, s, h, rows = op().fp8_norm_quant(x, w, 0.0, res, True)
    assert rows[0].isnan().all()  # 0 / 0
    q, s, h, rows = op().fp8_norm_quant(x, w, 1e-6, res, True)
    assert (q[0].float() == 0).all() and (rows[0] == 0).all()
    assert q[2].float().isnan().all() and s[2].isnan().all()
    assert rows[3, 200].isnan() and (rows[3, :200] == 0).all()
    for r in (1, 4):
        assert torch.equal(q[r].float(), want[0][r].float()) and torch.equal(rows[r], want[3][r])


# ------------------------------------------------------------------------ swiglu

SWIGLU_SLACK = 16 * U  # exp2 and the quotient are within 2 ulp, its argument's correction and the products half one each


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,limit", [(1, 16, 0.0), (3, 144, 0.0), (3, 144, 2.0), (2, 768, 7.0), (65, 2048, 0.0),
                                       (9, 14336, float("inf")), (1, 4112, 0.5)])
def test_swiglu_quant(m, n, limit, dtype):
    x = make_rows(m, 2 * n, n, dtype)
    q, s = op().fp8_swiglu_quant(x, limit)
    check_quant(q, s, swiglu64(x, 0.0 if limit == float("inf") else limit), SWIGLU_SLACK, f"{m} x {n}")
    wide = torch.full((m, 2 * n + 24), float("nan"), dtype=dtype, device="cuda")
    wide[:, 8:2 * n + 8] = x
    q2, s2 = op().fp8_swiglu_quant(wide[:, 8:2 * n + 8], limit)
    assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2)


def test_swiglu_every_gate():
    """Each finite gate alone in its group, so that the group's scale shows its value."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    g = bits[torch.isfinite(bits) & (bits.abs() < 1e30)]
    x = torch.zeros((len(g), 2, 16), dtype=BF)
    x[:, 0, 3], x[:, 1, 3] = g, 1.0
    q, s = op().fp8_swiglu_quant(x.view(-1, 32).cuda())
    want = swiglu64(x.view(-1, 32))[:, 3].abs().clamp(min=float(torch.tensor(1e-10))) / 448
    assert float(((s[:, 0].cpu().double() - want) / want).abs().max()) <= SWIGLU_SLACK


def test_swiglu_edges():
    inf, nan = float("inf"), float("nan")
    x = torch.zeros((7, 32), dtype=BF, device="cuda")
    x[0, 0], x[0, 16] = inf, 1.0
    x[1, 0], x[1, 16] = 1.0, nan
    x[2, 0], x[2, 16] = nan, 1.0
    x[3, 0], x[3, 16] = -3e38, 1.0
    x[4, 0], x[4, 16] = 3e38, 2.0
    x[5, 0], x[5, 16] = inf, -inf
    q, s = op().fp8_swiglu_quant(x, 0.0)
    assert s[0, 0] == inf and s[1:3].isnan().all() and s[4, 0] == inf and s[5, 0] == inf
    assert (q[3].float() == 0).all() and (q[6].float() == 0).all()
    q, s = op().fp8_swiglu_quant(x, 4.0)  # clamped infinities count as the limit, a NaN stays one
    v = swiglu64(torch.tensor([[4.0] + [0.0] * 15 + [1.0] + [0.0] * 15]))
    check_quant(q[:1].cpu(), s[:1].cpu(), v, SWIGLU_SLACK)
    check_quant(q[5:6].cpu(), s[5:6].cpu(), -4 * v, SWIGLU_SLACK)
    assert s[1:3].isnan().all()


# ----------------------------------------------------------------------- product

SHAPES = [(1, 16, 1), (1, 128, 128), (2, 144, 17), (5, 256, 576), (16, 1024, 130), (17, 528, 384), (31, 2048, 257),
          (33, 4096, 64), (64, 1040, 200), (65, 640, 96), (100, 384, 1000), (130, 512, 129), (257, 256, 640),
          (300, 1168, 515), (1, 14336, 512), (7, 16384, 48), (40, 14336, 256), (512, 2048, 768)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype,bias", [(BF, False), (HF, True)])
def test_linear(m, k, n, dtype, bias):
    print(f"case: linear m={m} k={k} n={n} {dtype} bias={bias}", flush=True)
    x = make_rows(m, k, m + n, dtype)
    w, ws = make_weight(n, k, n + k)
    b = make_rows(1, n, n, dtype)[0] if bias else None
    q, s = op().fp8_quant_rows(x)
    y = op().fp8_linear(q, w, ws, s, b, dtype == BF)
    assert y.dtype == dtype and y.shape == (m, n)
    check_product(y, q, s, w, ws, b, f"{m} {k} {n}")
    assert torch.equal(y, op().fp8_linear(q, w, ws, s, b, dtype == BF))
    # from the 16-bit rows: the same quantized rows
    check_product(op().fp8_linear(x, w, ws, None, b, dtype == BF), q, s, w, ws, b, f"rows {m} {k} {n}")


@pytest.mark.parametrize("m", [1, 3, 16, 40, 200])
def test_linear_types_shapes_and_strides(m):
    k, n = 400, 150
    x, (w, ws) = make_rows(m, k, 5, HF), make_weight(n, k, 6)
    q, s = op().fp8_quant_rows(x)
    want = op().fp8_linear(q, w, ws, s)
    check_product(want, q, s, w, ws)
    check_product(op().fp8_linear(x, w, ws, None, None, True), q, s, w, ws)  # fp16 rows, bf16 result
    odd = torch.zeros(m * k + 1, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[1:].view(m, k)
    odd.copy_(q)
    wide = torch.zeros((n, k + 16), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wide[:, :k].copy_(w)
    scale = torch.zeros((s.shape[1], m), device="cuda")
    scale.copy_(s.t())
    for args in ((odd, w, ws, s), (q, wide[:, :k], ws, s), (q, w, ws.t().contiguous().t(), scale.t()),
                 (q.view(1, m, k), w, ws, s.view(1, m, -1))):
        assert torch.equal(op().fp8_linear(*args), want)
    assert op().fp8_linear(q[:0], w, ws, s[:0]).shape == (0, n)
    assert op().fp8_linear(x[:0], w, ws).shape == (0, n)


@pytest.mark.parametrize("m", [1, 4, 40, 300])
def test_linear_bad_values_stay_in_their_row(m):
    """A NaN or infinity in a row makes that row's outputs NaN and no others; one in a weight, its column's."""
    k, n = 272, 200
    x, (w, ws) = make_rows(m, k, 7), make_weight(n, k, 8)
    r = m // 2
    x[r, 270] = float("inf")
    y = op().fp8_linear(x, w, ws)
    assert y[r].isnan().all() and torch.cat((y[:r], y[r + 1:])).isfinite().all()
    x[r, 270] = 1.0
    w.view(torch.uint8)[131, 5] = 0x7F
    y = op().fp8_linear(x, w, ws)
    assert y[:, 131].isnan().all() and torch.cat((y[:, :131], y[:, 132:]), 1).isfinite().all()
    w.view(torch.uint8)[131, 5] = 0
    ws[1, 2] = float("nan")
    y = op().fp8_linear(x, w, ws)
    assert y[:, 128:].isnan().all() and y[:, :128].isfinite().all()


def test_linear_writes_only_its_output(monkeypatch):
    """What lies behind y is left as it was, at ragged sizes, and so is what lies around the inputs."""
    import ctypes

    from sglang_exl3 import _lib

    for m, k, n in ((1, 128, 1), (1, 256, 130), (19, 144, 131), (70, 272, 67), (260, 256, 259)):
        x, (w, ws) = make_rows(m, k, 1), make_weight(n, k, 2)
        q, s = op().fp8_quant_rows(x)
        y = torch.full((m * n + 256,), 7.0, dtype=BF, device="cuda")
        buf = torch.zeros(int(_lib.lib().exl3_fp8_linear_workspace_size(_lib.DTYPE_E4M3, m, k, n)) or 256,
                          dtype=torch.uint8, device="cuda")
        rc = _lib.lib().exl3_fp8_linear(q.data_ptr(), _lib.DTYPE_E4M3, s.data_ptr(), w.data_ptr(), ws.data_ptr(), None,
                                        y.data_ptr(), _lib.DTYPE_BF16, m, k, n, buf.data_ptr(), buf.numel(),
                                        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        assert (y[m * n:] == 7).all()
        check_product(y[:m * n].view(m, n), q, s, w, ws)


# ------------------------------------------------------------ together, as they are used

def _mlp(x, res, gain, gu, down, limit=0.0):
    q, s, h = op().fp8_norm_quant(x, gain, 1e-6, res)
    q, s = op().fp8_swiglu_quant(op().fp8_linear(q, *gu, s), limit)
    return op().fp8_linear(q, *down, s), h


def _mlp_inputs(m, k, n, seed):
    gain = torch.ones(k, dtype=BF, device="cuda")
    return (make_rows(m, k, seed), make_rows(m, k, seed + 1), gain, make_weight(2 * n, k, seed + 2),
            make_weight(k, n, seed + 3))


@pytest.mark.parametrize("m,k,n", [(1, 256, 384), (3, 2048, 768), (40, 512, 1040), (150, 400, 272)])
def test_mlp(m, k, n):
    """Each step against 64 bits from what the step before returned."""
    x, res, gain, gu, down = _mlp_inputs(m, k, n, m)
    q, s, h = op().fp8_norm_quant(x, gain, 1e-6, res)
    check_quant(q, s, norm64(x, gain, 1e-6, res)[1], norm_slack(k) + 2 * U)
    y = op().fp8_linear(q, *gu, s)
    check_product(y, q, s, *gu)
    q, s = op().fp8_swiglu_quant(y)
    check_quant(q, s, swiglu64(y), SWIGLU_SLACK)
    z = op().fp8_linear(q, *down, s)
    check_product(z, q, s, *down)
    got = _mlp(x, res, gain, gu, down)
    assert torch.equal(got[0], z) and torch.equal(got[1], h)


@pytest.mark.parametrize("m", [1, 24, 200])
def test_mlp_in_a_graph(m):
    """A captured pass replayed on new inputs, eager calls on the same stream between the replays."""
    k, n = 512, 640
    x, res, gain, gu, down = _mlp_inputs(m, k, n, 77)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        def both():
            y, h = _mlp(x, res, gain, gu, down)
            return y, h, op().fp8_linear(x, *gu)
        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = both()
        for seed in range(4):
            x.copy_(make_rows(m, k, 100 + seed))
            res.copy_(make_rows(m, k, 200 + seed))
            want = both()
            st.synchronize()
            graph.replay()
            st.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(st)


def test_two_streams_at_once():
    """Calls in flight on two streams have a workspace each."""
    k, n = 2048, 512
    w, ws = make_weight(n, k, 1)
    xs = [make_rows(40, k, s) for s in (1, 2)]
    want = [op().fp8_linear(x, w, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(op().fp8_linear(xs[i], w, ws))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])


# -------------------------------------------------------------------- the layer

@pytest.mark.parametrize("m", [1, 20, 150])
def test_layer_from_a_checkpoint(m):
    """qkv of three shards loaded one by one through the layer's loaders, applied to rows and to quantized rows."""
    from torch import nn

    from sglang_exl3.exl3 import EXL3Config
    from sglang_exl3.fp8 import FP8BlockLinearMethod

    class QKVParallelLinear(nn.Module):
        pass

    cfg = EXL3Config.from_config({"quant_method": "exl3", "bits": 3, "scope": "glm53_routed_experts_only",
                                  "non_routed_quantization": {"quant_method": "fp8", "weight_block_size": [128, 128],
                                                              "activation_scheme": "dynamic"}})
    layer = QKVParallelLinear()
    method = cfg.get_quant_method(layer, "model.layers.0.self_attn.qkv_proj")
    assert isinstance(method, FP8BlockLinearMethod)
    k, widths = 640, [512, 128, 72]
    method.create_weights(layer, k, widths, k, sum(widths), BF)
    shards = [make_weight(n, k, n) for n in widths]
    layer.cuda()
    for name, (w, ws) in zip("qkv", shards):
        layer.weight.weight_loader(layer.weight, w.cpu(), name)
        layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, ws.cpu(), name)
    method.process_weights_after_loading(layer)
    x = make_rows(m, k, 4)
    q, s = op().fp8_quant_rows(x)
    bias = make_rows(1, sum(widths), 3)[0]
    y = method.apply(layer, x.view(1, m, k), bias)
    assert y.shape == (1, m, sum(widths)) and y.dtype == BF
    w, ws = torch.cat([a for a, _ in shards]), torch.cat([b for _, b in shards])
    check_product(y[0], q, s, w, ws, bias)
    check_product(method.apply(layer, (q, s), bias), q, s, w, ws, bias)
    check_product(method.apply(layer, x.float()), q, s, w, ws)


# --------------------------------------------------------------------- refusals

def test_refusals_on_the_device():
    x, (w, ws) = make_rows(4, 256, 1), make_weight(128, 256, 2)
    q, s = op().fp8_quant_rows(x)
    g = torch.ones(256, dtype=BF, device="cuda")
    bad = [
        (lambda: op().fp8_quant_rows(x.float()), "float16 or bfloat16"),
        (lambda: op().fp8_quant_rows(x[:, :24].contiguous()), "multiple of 16"),
        (lambda: op().fp8_quant_rows(x[0, 0]), "shape"),
        (lambda: op().fp8_norm_quant(x, g[:128], 1e-6), "weight must be"),
        (lambda: op().fp8_norm_quant(x, g.half(), 1e-6), "weight must be"),
        (lambda: op().fp8_norm_quant(x, g, 1e-6, x[:2]), "residual must be"),
        (lambda: op().fp8_norm_quant(x, g, -1.0), "eps"),
        (lambda: op().fp8_norm_quant(x, g, float("nan")), "eps"),
        (lambda: op().fp8_norm_quant(torch.zeros((1, 32784), dtype=BF, device="cuda"),
                                     torch.zeros(32784, dtype=BF, device="cuda"), 1e-6), "above 32768"),
        (lambda: op().fp8_swiglu_quant(x, -1.0), "nonnegative"),
        (lambda: op().fp8_swiglu_quant(x[:, :48].contiguous(), 0.0), "multiple of 16"),
        (lambda: op().fp8_linear(x[:, :128], w, ws), "x must have shape"),
        (lambda: op().fp8_linear(x, w.float(), ws), "float8_e4m3fn"),
        (lambda: op().fp8_linear(x, w, ws[:, :1]), "weight_scale must be"),
        (lambda: op().fp8_linear(x, w, ws.half()), "weight_scale must be"),
        (lambda: op().fp8_linear(q, w, ws), "x_scale"),
        (lambda: op().fp8_linear(q, w, ws, s[:, :1]), "x_scale"),
        (lambda: op().fp8_linear(x, w, ws, s), "x_scale goes with"),
        (lambda: op().fp8_linear(x.float(), w, ws), "x must be"),
        (lambda: op().fp8_linear(x, w, ws, None, torch.zeros(128, device="cuda")), "bias must be"),
        (lambda: op().fp8_linear(x, w, ws, None, torch.zeros(64, dtype=BF, device="cuda")), "bias must be"),
        (lambda: op().fp8_linear(x, w, ws.cpu()), "HIP device"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
